// Group norm with an activation, channels last, sm_100a: forward and gradient.
//
// x [N, S, C], G groups of Cg = C/G channels; statistics of (n, g) over its S*Cg values:
//   xh = (x - mean) rstd,  z = xh w_c + b_c,  y = act(z)      (act: none or z sigmoid(z))
//   dz = dy act'(z),  dw_c = sum_{n,s} dz xh,  db_c = sum_{n,s} dz,  e = dz w_c
//   dx = rstd (e - mean_g(e) - xh mean_g(e xh))
// S = 1 is the Block's norm of each head and token (hdcmamba/model.py:285-292).
// Statistics and sums are fp32; y, dx, dw, db are rounded once to their types.
//
// Schedules (bound by HBM: x read and y written; x, dy read and dx written):
//   * one position (S = 1): a group is Cg neighbouring values.  A few lanes (LG, a power of two)
//     hold one group of one sample in registers, with its mean, its centred squares (or the two
//     sums of the gradient) summed by shuffles; a CTA covers whole samples, and a thread keeps its
//     channels from sample to sample, so that weight and bias stay in registers and dw and db
//     accumulate there.  One pass over the data.
//   * otherwise two passes: a CTA takes a slice of a sample's positions, a thread a few channels
//     of every RL-th of them.  First each slice's statistics (or sums of the gradient), then, with
//     the slices of a sample joined in their order, the outputs; the second reading of the
//     input comes from L2 where it fits (126 MB).
// Statistics never cancel: a thread takes blocks of rows, each with its own mean and centred
// squares, and blocks, threads and slices are joined by
//   n = n1 + n2, mean = mean1 + (mean2 - mean1) n2/n, M2 = M2_1 + M2_2 + (mean2 - mean1)^2 n1 n2/n.
// Channels per load: as many as 16 bytes hold and the row (S = 1: the group) divides into.
// Measured (device time, against 6550 GB/s): 16 x 4096 x 320 bf16 forward 34 us (38%): statistics
// 16, joining 3, outputs 15, each bound by the latency of its loads at 24 warps per SM;
// 4 x 16384 x 128 fp32 forward 25 us (40%), backward 46 us (33%); 2 x 225 x 96 bf16 6.2 and 7.5 us.
#include "group_norm.cuh"

namespace hdc {

// ---------------------------------------------------------------- several positions per sample
// CTA (sample and slice, channel block): thread = (row lane, chunk of VE channels).
constexpr int kGnThreads = 256;
// resident CTAs per SM of the two-pass kernels (forward with four: 39 us for 34, 16 x 4096 x 320)
constexpr int kGnFwdCtas = 3, kGnBwdCtas = 2;
// row lanes of a CTA: threads per chunk of channels (one when a thread has several chunks)
__host__ __device__ inline int gn_lanes(int nchunk) { return nchunk < kGnThreads ? kGnThreads / nchunk : 1; }

// A CTA's place: sample n, slice of its positions from r0 (rows of them), channels c_lo .. c_lo + cw
struct GnPlace {
  int n, slice, r0, rows, c_lo, cw;
  __device__ explicit GnPlace(const GnParams& p) {
    n = blockIdx.x / p.slices;
    slice = blockIdx.x - n * p.slices;
    r0 = slice * p.rows;
    rows = min(p.rows, p.S - r0);
    c_lo = blockIdx.y * p.cb;
    cw = min(p.cb, p.C - c_lo);
  }
};

// neg = -mean and rstd of the channels c0 .. c0 + VE - 1, from arrays indexed by group
template <int VE>
__device__ __forceinline__ void gn_groups(const float* mean, const float* rstd, int c0, int Cg, Fv<VE>& neg, Fv<VE>& rs) {
  int g = c0 / Cg, end = (g + 1) * Cg;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    if (c0 + i >= end) ++g, end += Cg;
    neg.v[i] = -mean[g];
    rs.v[i] = rstd[g];
  }
}

// The slice's outputs; mean and rstd indexed by the block's groups.
template <typename T, int VE, bool WHOLE>
__device__ __forceinline__ void gn_apply_rows(const GnParams& p, const GnPlace& at, const float* gmean, const float* grstd) {
  const int nchunk = at.cw / VE, RL = gn_lanes(nchunk), per = min(nchunk, kGnThreads), rl = threadIdx.x / per;
  if (rl >= RL) return;
  for (int k = threadIdx.x - rl * per; k < nchunk; k += per) {
    const int c0 = at.c_lo + k * VE;
    const Fv<VE> w = gn_params<VE>(p.w, p.p_bf16, c0, 1.f), b = gn_params<VE>(p.b, p.p_bf16, c0, 0.f);
    wait_for_previous();
    Fv<VE> neg, sc;
    gn_groups<VE>(gmean, grstd, k * VE, p.Cg, neg, sc);
    sc = sc * w;
    const T* x = static_cast<const T*>(p.x) + at.n * p.xsn + (int64_t)(at.r0 + rl) * p.xss + c0;
    T* y = static_cast<T*>(p.y) + at.n * p.ysn + (int64_t)(at.r0 + rl) * p.yss + c0;
    const int64_t xh = RL * p.xss, yh = RL * p.yss;
    constexpr int U = 4;
    int r = rl;
    for (; r + (U - 1) * RL < at.rows; r += U * RL) {
      Raw<T, VE> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = ld_raw<T, VE, WHOLE, true>(x + u * xh);
      x += U * xh;
#pragma unroll
      for (int u = 0; u < U; ++u)
        st_vec<T, VE, WHOLE>(y + u * yh, gn_act<T>(fma(unpack<T, VE>(raw[u]) + neg, sc, b), p.silu));
      y += U * yh;
    }
    for (; r < at.rows; r += RL, x += xh, y += yh)
      st_vec<T, VE, WHOLE>(y, gn_act<T>(fma(unpack<T, VE>(ld_raw<T, VE, WHOLE, true>(x)) + neg, sc, b), p.silu));
  }
}

// (mean, M2) of each slice and group; ONE (a single slice): mean and rstd, and the outputs too,
// the second reading from L1 or L2.
template <typename T, int VE, bool WHOLE, bool ONE>
__global__ void __launch_bounds__(kGnThreads, kGnFwdCtas) gn_stats_kernel(const __grid_constant__ GnParams p) {
  extern __shared__ float sh[];  // [2][row lanes][cw]: mean, M2; ONE: [2][groups]
  const GnPlace at(p);
  const int nchunk = at.cw / VE, RL = gn_lanes(nchunk), per = min(nchunk, kGnThreads), rl = threadIdx.x / per;
  constexpr int U = 4;
  let_next_start();
  if (rl < RL)
    for (int k = threadIdx.x - rl * per; k < nchunk; k += per) {
      const T* x = static_cast<const T*>(p.x) + at.n * p.xsn + (int64_t)(at.r0 + rl) * p.xss + at.c_lo + k * VE;
      const int64_t hop = RL * p.xss;
      Fv<VE> mean = all<VE>(0.f), M2 = all<VE>(0.f);
      float blocks = 0.f;  // of U rows
      int r = rl;
      Raw<T, VE> raw[U];
      auto load = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = ld_raw<T, VE, WHOLE, true>(x + u * hop);
        x += U * hop;
      };
      bool more = r + (U - 1) * RL < at.rows;
      if (more) load();
      while (more) {
        Fv<VE> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = unpack<T, VE>(raw[u]);
        r += U * RL;
        more = r + (U - 1) * RL < at.rows;
        if (more) load();
        Fv<VE> m = (v[0] + v[1]) + (v[2] + v[3]);
        m = m * all<VE>(1.f / U);
        const Fv<VE> neg = m * all<VE>(-1.f);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const Fv<VE> d = v[u] + neg;
          M2 = fma(d, d, M2);
        }
        blocks += 1.f;
        const float f = rcp(blocks);  // off by 2^-23: the mean by that much of a block's deviation
        const Fv<VE> d = fma(mean, all<VE>(-1.f), m);
        mean = fma(d, all<VE>(f), mean);
        M2 = fma(d * d, all<VE>(U * (blocks - 1.f) * f), M2);
      }
      float cnt = blocks * U;
      for (; r < at.rows; r += RL) {
        const Fv<VE> d = fma(mean, all<VE>(-1.f), unpack<T, VE>(ld_raw<T, VE, WHOLE, true>(x)));
        x += hop;
        const float f = rcp(cnt + 1.f);
        mean = fma(d, all<VE>(f), mean);
        M2 = fma(d * d, all<VE>(cnt * f), M2);
        cnt += 1.f;
      }
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        sh[rl * at.cw + k * VE + i] = mean.v[i];
        sh[(RL + rl) * at.cw + k * VE + i] = M2.v[i];
      }
    }
  __syncthreads();
  // channels over the row lanes (lane q has the rows q, q + RL, ...)
  const int lanes = min(RL, at.rows), base = at.rows / RL, extra = at.rows - base * RL;
  const float nr = (float)at.rows, n0 = (float)base, n1 = (float)(base + 1);
  for (int c = threadIdx.x; c < at.cw; c += kGnThreads) {
    float m = 0.f;
    for (int q = 0; q < lanes; ++q) m = fmaf(q < extra ? n1 : n0, sh[q * at.cw + c], m);
    m = over(m, nr, 1.f / nr);
    float M2 = 0.f;
    for (int q = 0; q < lanes; ++q) {
      const float d = sh[q * at.cw + c] - m;
      M2 += fmaf((q < extra ? n1 : n0) * d, d, sh[(RL + q) * at.cw + c]);
    }
    sh[c] = m;  // only this thread reads and writes this channel here
    sh[RL * at.cw + c] = M2;
  }
  __syncthreads();
  // groups over their channels: a few lanes each
  const int ng = at.cw / p.Cg;
  const float nc = (float)p.Cg, invc = 1.f / nc;
  int lg = 1;
  while (lg < 32 && lg < p.Cg) lg *= 2;
  const int l = threadIdx.x & (lg - 1);
  float* gmean = sh + 2 * RL * at.cw;
  for (int g0 = 0; g0 < ng; g0 += kGnThreads / lg) {
    const int gi = g0 + threadIdx.x / lg;
    const float* m = sh + min(gi, ng - 1) * p.Cg;
    float mean = 0.f, M2 = 0.f;
    for (int c = l; c < p.Cg; c += lg) mean += m[c];
    for (int o = lg / 2; o > 0; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    mean = over(mean, nc, invc);
    for (int c = l; c < p.Cg; c += lg) {
      const float d = m[c] - mean;
      M2 += fmaf(nr * d, d, m[RL * at.cw + c]);
    }
    for (int o = lg / 2; o > 0; o >>= 1) M2 += __shfl_xor_sync(0xffffffffu, M2, o);
    if (l == 0 && gi < ng) {
      if constexpr (ONE) {
        const float rstd = gn_rstd(M2, invc / nr, p.eps);
        gmean[gi] = mean;
        gmean[ng + gi] = rstd;
        if (p.mean) {
          p.mean[(int64_t)at.n * p.G + at.c_lo / p.Cg + gi] = mean;
          p.rstd[(int64_t)at.n * p.G + at.c_lo / p.Cg + gi] = rstd;
        }
      } else {
        p.stats[(int64_t)blockIdx.x * p.G + at.c_lo / p.Cg + gi] = make_float2(mean, M2);
      }
    }
  }
  if constexpr (ONE) {
    __syncthreads();
    gn_apply_rows<T, VE, WHOLE>(p, at, gmean, gmean + ng);
  }
}

// mean and rstd of each (n, g) from its slices: one warp each
__global__ void __launch_bounds__(256) gn_join_kernel(const __grid_constant__ GnParams p) {
  let_next_start();
  wait_for_previous();
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= (int64_t)p.N * p.G) return;
  const int n = (int)(i / p.G), g = (int)(i - (int64_t)n * p.G);
  const float2* st = p.stats + (int64_t)n * p.slices * p.G + g;
  const float total = (float)p.S * (float)p.Cg;
  float mean = 0.f;
  for (int q = lane; q < p.slices; q += 32)
    mean = fmaf((float)min(p.rows, p.S - q * p.rows) * (float)p.Cg, st[(int64_t)q * p.G].x, mean);
  mean = warp_sum(mean) / total;
  float M2 = 0.f;
  for (int q = lane; q < p.slices; q += 32) {
    const float2 v = st[(int64_t)q * p.G];
    const float d = v.x - mean;
    M2 += fmaf((float)min(p.rows, p.S - q * p.rows) * (float)p.Cg * d, d, v.y);
  }
  M2 = warp_sum(M2);
  if (lane == 0) {
    p.mean[i] = mean;
    p.rstd[i] = gn_rstd(M2, 1.f / total, p.eps);
  }
}

template <typename T, int VE, bool WHOLE>
__global__ void __launch_bounds__(kGnThreads, kGnFwdCtas) gn_apply_kernel(const __grid_constant__ GnParams p) {
  const GnPlace at(p);
  const int64_t g0 = (int64_t)at.n * p.G + at.c_lo / p.Cg;
  gn_apply_rows<T, VE, WHOLE>(p, at, p.mean + g0, p.rstd + g0);
}

// The slice's dx; the means of e xh and of e indexed by the block's groups.
template <typename T, int VE, bool WHOLE>
__device__ __forceinline__ void gn_dx_rows(const GnParams& p, const GnPlace& at, const float* mx, const float* me) {
  const int nchunk = at.cw / VE, RL = gn_lanes(nchunk), per = min(nchunk, kGnThreads), rl = threadIdx.x / per;
  if (rl >= RL) return;
  const int64_t g0 = (int64_t)at.n * p.G + at.c_lo / p.Cg;
  for (int k = threadIdx.x - rl * per; k < nchunk; k += per) {
    const int c0 = at.c_lo + k * VE;
    const Fv<VE> w = gn_params<VE>(p.w, p.p_bf16, c0, 1.f), b = gn_params<VE>(p.b, p.p_bf16, c0, 0.f);
    Fv<VE> neg, rstd, sx, se;
    gn_groups<VE>(p.mean + g0, p.rstd + g0, k * VE, p.Cg, neg, rstd);
    wait_for_previous();
    gn_groups<VE>(mx, me, k * VE, p.Cg, sx, se);
    se = se * all<VE>(-1.f);
    const T* x = static_cast<const T*>(p.x) + at.n * p.xsn + (int64_t)(at.r0 + rl) * p.xss + c0;
    const T* dy = static_cast<const T*>(p.dy) + at.n * p.dsn + (int64_t)(at.r0 + rl) * p.dss + c0;
    T* dx = static_cast<T*>(p.dx) + at.n * p.gsn + (int64_t)(at.r0 + rl) * p.gss + c0;
    const int64_t xh = RL * p.xss, dh = RL * p.dss, gh = RL * p.gss;
    auto one = [&](const Raw<T, VE>& xr, const Raw<T, VE>& dr, T* to) {
      const Fv<VE> v = (unpack<T, VE>(xr) + neg) * rstd;
      const Fv<VE> dz = gn_dact<T>(unpack<T, VE>(dr), fma(v, w, b), p.silu);
      st_vec<T, VE, WHOLE>(to, fma(v, sx, fma(dz, w, se)) * rstd);
    };
    constexpr int U = 4;
    int r = rl;
    for (; r + (U - 1) * RL < at.rows; r += U * RL) {
      Raw<T, VE> xr[U], dr[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        xr[u] = ld_raw<T, VE, WHOLE, false>(x + u * xh);
        dr[u] = ld_raw<T, VE, WHOLE, false>(dy + u * dh);
      }
      x += U * xh, dy += U * dh;
#pragma unroll
      for (int u = 0; u < U; ++u) one(xr[u], dr[u], dx + u * gh);
      dx += U * gh;
    }
    for (; r < at.rows; r += RL, x += xh, dy += dh, dx += gh)
      one(ld_raw<T, VE, WHOLE, false>(x), ld_raw<T, VE, WHOLE, false>(dy), dx);
  }
}

// The gradient's sums per channel of each slice: part[n * slices + slice][2][C]; ONE: dx too.
template <typename T, int VE, bool WHOLE, bool ONE>
__global__ void __launch_bounds__(kGnThreads, kGnBwdCtas) gn_sums_kernel(const __grid_constant__ GnParams p) {
  extern __shared__ float sh[];  // [2][row lanes][cw]; ONE: [2][cw], [2][groups]
  const GnPlace at(p);
  const int nchunk = at.cw / VE, RL = gn_lanes(nchunk), per = min(nchunk, kGnThreads), rl = threadIdx.x / per;
  const int64_t g0 = (int64_t)at.n * p.G + at.c_lo / p.Cg;
  let_next_start();
  if (rl < RL)
    for (int k = threadIdx.x - rl * per; k < nchunk; k += per) {
      const int c0 = at.c_lo + k * VE;
      const Fv<VE> w = gn_params<VE>(p.w, p.p_bf16, c0, 1.f), b = gn_params<VE>(p.b, p.p_bf16, c0, 0.f);
      Fv<VE> neg, rstd, a0 = all<VE>(0.f), a1 = all<VE>(0.f);
      gn_groups<VE>(p.mean + g0, p.rstd + g0, k * VE, p.Cg, neg, rstd);
      const T* x = static_cast<const T*>(p.x) + at.n * p.xsn + (int64_t)(at.r0 + rl) * p.xss + c0;
      const T* dy = static_cast<const T*>(p.dy) + at.n * p.dsn + (int64_t)(at.r0 + rl) * p.dss + c0;
      const int64_t xh = RL * p.xss, dh = RL * p.dss;
      auto one = [&](const Raw<T, VE>& xr, const Raw<T, VE>& dr) {
        const Fv<VE> v = (unpack<T, VE>(xr) + neg) * rstd;
        const Fv<VE> dz = gn_dact<T>(unpack<T, VE>(dr), fma(v, w, b), p.silu);
        a0 = fma(dz, v, a0);
        a1 = a1 + dz;
      };
      constexpr int U = 4;
      int r = rl;
      for (; r + (U - 1) * RL < at.rows; r += U * RL) {
        Raw<T, VE> xr[U], dr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          xr[u] = ld_raw<T, VE, WHOLE, !ONE>(x + u * xh);
          dr[u] = ld_raw<T, VE, WHOLE, !ONE>(dy + u * dh);
        }
        x += U * xh, dy += U * dh;
#pragma unroll
        for (int u = 0; u < U; ++u) one(xr[u], dr[u]);
      }
      for (; r < at.rows; r += RL, x += xh, dy += dh) one(ld_raw<T, VE, WHOLE, !ONE>(x), ld_raw<T, VE, WHOLE, !ONE>(dy));
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        sh[rl * at.cw + k * VE + i] = a0.v[i];
        sh[(RL + rl) * at.cw + k * VE + i] = a1.v[i];
      }
    }
  __syncthreads();
  float* tot = sh + 2 * RL * at.cw;
  for (int i = threadIdx.x; i < 2 * at.cw; i += kGnThreads) {
    const int which = i >= at.cw, c = which ? i - at.cw : i;
    float v = 0.f;
    for (int q = 0; q < RL; ++q) v += sh[(which * RL + q) * at.cw + c];
    p.part[((int64_t)blockIdx.x * 2 + which) * p.C + at.c_lo + c] = v;
    if constexpr (ONE) tot[i] = v * gn_param(p.w, p.p_bf16, at.c_lo + c, 1.f);
  }
  if constexpr (ONE) {
    __syncthreads();
    const int lane = threadIdx.x & 31, ng = at.cw / p.Cg;
    float* gm = tot + 2 * at.cw;
    const float inv = 1.f / ((float)p.S * (float)p.Cg);
    for (int i = threadIdx.x >> 5; i < 2 * ng; i += kGnThreads / 32) {
      const int which = i >= ng, gi = which ? i - ng : i;
      float v = 0.f;
      for (int c = lane; c < p.Cg; c += 32) v += tot[which * at.cw + gi * p.Cg + c];
      v = warp_sum(v);
      if (lane == 0) gm[i] = v * inv;
    }
    __syncthreads();
    gn_dx_rows<T, VE, WHOLE>(p, at, gm, gm + ng);
  }
}

// CTA (sample, block of whole groups): the sample's sums over its slices, to sums[n][2][C], and
// from them the means of e xh and of e of each group, to gmean[n][2][G].
__global__ void __launch_bounds__(256) gn_mid_kernel(const __grid_constant__ GnParams p, int block) {
  extern __shared__ float sh[];  // [strands][2 cw]; then the sums times the weight in the first of them
  let_next_start();
  wait_for_previous();
  const int n = blockIdx.x, c_lo = blockIdx.y * block, cw = min(block, p.C - c_lo), items = 2 * cw;
  const int per = min(items, 256), strands = 256 / per, st = threadIdx.x / per;
  if (st < strands)
    for (int i = threadIdx.x - st * per; i < items; i += per) {
      const int which = i >= cw, c = which ? i - cw : i;
      const float* q = p.part + ((int64_t)n * p.slices * 2 + which) * p.C + c_lo + c;
      float v = 0.f;
#pragma unroll 8
      for (int k = st; k < p.slices; k += strands) v += q[(int64_t)k * 2 * p.C];
      sh[st * items + i] = v;
    }
  __syncthreads();
  float* tot = sh;
  for (int i = threadIdx.x; i < items; i += 256) {  // item i of every strand is this thread's alone
    float v = sh[i];
    for (int k = 1; k < strands; ++k) v += sh[k * items + i];
    const int which = i >= cw, c = which ? i - cw : i;
    p.sums[((int64_t)n * 2 + which) * p.C + c_lo + c] = v;
    tot[i] = v * gn_param(p.w, p.p_bf16, c_lo + c, 1.f);
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, ng = cw / p.Cg;
  const float inv = 1.f / ((float)p.S * (float)p.Cg);
  for (int i = threadIdx.x >> 5; i < 2 * ng; i += 8) {
    const int which = i >= ng, gi = which ? i - ng : i;
    float v = 0.f;
    for (int c = lane; c < p.Cg; c += 32) v += tot[which * cw + gi * p.Cg + c];
    v = warp_sum(v);
    if (lane == 0) p.gmean[((int64_t)n * 2 + which) * p.G + c_lo / p.Cg + gi] = v * inv;
  }
}

template <typename T, int VE, bool WHOLE>
__global__ void __launch_bounds__(kGnThreads, kGnBwdCtas) gn_dx_kernel(const __grid_constant__ GnParams p) {
  const GnPlace at(p);
  const int64_t g0 = (int64_t)at.n * 2 * p.G + at.c_lo / p.Cg;
  gn_dx_rows<T, VE, WHOLE>(p, at, p.gmean + g0, p.gmean + g0 + p.G);
}

// ---------------------------------------------------------------- groups of more than 4096 channels
// One CTA per (n, g), the group read again for each of its sums.
__device__ __forceinline__ float block_sum(float v) {
  __shared__ float red[8];
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int k = 0; k < 8; ++k) s += red[k];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(256) gn_any_fwd_kernel(GnParams p) {
  const int n = blockIdx.x / p.G, g = blockIdx.x - n * p.G;
  const T* x = static_cast<const T*>(p.x) + n * p.xsn + g * p.Cg;
  T* y = static_cast<T*>(p.y) + n * p.ysn + g * p.Cg;
  const int64_t M = (int64_t)p.S * p.Cg;
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < M; i += 256) s += to_f(x[(i / p.Cg) * p.xss + i % p.Cg]);
  const float mean = block_sum(s) / (float)M;
  s = 0.f;
  for (int64_t i = threadIdx.x; i < M; i += 256) {
    const float d = to_f(x[(i / p.Cg) * p.xss + i % p.Cg]) - mean;
    s = fmaf(d, d, s);
  }
  const float rstd = rsqrtf(block_sum(s) / (float)M + p.eps);
  if (threadIdx.x == 0 && p.mean) {
    p.mean[blockIdx.x] = mean;
    p.rstd[blockIdx.x] = rstd;
  }
  for (int64_t i = threadIdx.x; i < M; i += 256) {
    const int c = (int)(i % p.Cg);
    const int64_t r = i / p.Cg;
    const float xh = (to_f(x[r * p.xss + c]) - mean) * rstd;
    const float z = fmaf(xh, gn_param(p.w, p.p_bf16, g * p.Cg + c, 1.f), gn_param(p.b, p.p_bf16, g * p.Cg + c, 0.f));
    y[r * p.yss + c] = from_f<T>(p.silu ? z / (1.f + expf(-z)) : z);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) gn_any_bwd_kernel(GnParams p) {
  const int n = blockIdx.x / p.G, g = blockIdx.x - n * p.G;
  const T* x = static_cast<const T*>(p.x) + n * p.xsn + g * p.Cg;
  const T* dy = static_cast<const T*>(p.dy) + n * p.dsn + g * p.Cg;
  T* dx = static_cast<T*>(p.dx) + n * p.gsn + g * p.Cg;
  const float mean = p.mean[blockIdx.x], rstd = p.rstd[blockIdx.x];
  auto grad = [&](int64_t r, int c, float& xh, float w, float b) {
    xh = (to_f(x[r * p.xss + c]) - mean) * rstd;
    float dz = to_f(dy[r * p.dss + c]);
    if (p.silu) {
      const float z = fmaf(xh, w, b), q = 1.f / (1.f + expf(-z));
      dz *= q * (1.f + z * (1.f - q));
    }
    return dz;
  };
  float se = 0.f, sx = 0.f;  // sums over the group of e and e xh
  for (int c = 0; c < p.Cg; ++c) {
    const float w = gn_param(p.w, p.p_bf16, g * p.Cg + c, 1.f), b = gn_param(p.b, p.p_bf16, g * p.Cg + c, 0.f);
    float a0 = 0.f, a1 = 0.f;
    for (int r = threadIdx.x; r < p.S; r += 256) {
      float xh;
      const float dz = grad(r, c, xh, w, b);
      a0 = fmaf(dz, xh, a0);
      a1 += dz;
    }
    a0 = block_sum(a0);
    a1 = block_sum(a1);
    if (threadIdx.x == 0) {
      p.part[((int64_t)n * 2) * p.C + g * p.Cg + c] = a0;
      p.part[((int64_t)n * 2 + 1) * p.C + g * p.Cg + c] = a1;
    }
    se = fmaf(w, a1, se);
    sx = fmaf(w, a0, sx);
  }
  const int64_t M = (int64_t)p.S * p.Cg;
  se /= (float)M;
  sx /= (float)M;
  for (int64_t i = threadIdx.x; i < M; i += 256) {
    const int c = (int)(i % p.Cg);
    const int64_t r = i / p.Cg;
    const float w = gn_param(p.w, p.p_bf16, g * p.Cg + c, 1.f), b = gn_param(p.b, p.p_bf16, g * p.Cg + c, 0.f);
    float xh;
    const float dz = grad(r, c, xh, w, b);
    dx[r * p.gss + c] = from_f<T>(rstd * (fmaf(dz, w, -se) - xh * sx));
  }
}

// dw[c] (blockIdx.y 0) and db[c] (1): sums of the parts, 32 strands per channel, then the strands
__global__ void __launch_bounds__(1024) gn_param_grad_kernel(const float* part, int64_t parts, int C, void* dw, void* db,
                                                             int bf16) {
  __shared__ float s[32][33];
  const int x = threadIdx.x & 31, k = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  void* out = blockIdx.y ? db : dw;
  wait_for_previous();
  if (!out) return;
  float v = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int64_t i = k; i < parts; i += 32) v += part[(i * 2 + blockIdx.y) * C + c];
  }
  s[k][x] = v;
  __syncthreads();
  if (k != 0 || c >= C) return;
  for (int i = 1; i < 32; ++i) v += s[i][x];
  if (bf16) static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(v);
  else static_cast<float*>(out)[c] = v;
}

// ---------------------------------------------------------------- plans
constexpr int kGnMostCg = 4096;  // channels of a group in the kernels above
// SMs that the schedules fill: B200's, as a constant, so that the sizes of the workspaces and the
// order of the sums are a matter of the shape alone
constexpr int kGnSms = 148;

static GnRowPlan gn_row_plan(int64_t N, int64_t S, int64_t G, int64_t Cg, int ve, bool bwd = false) {
  GnRowPlan r{};
  const int64_t chunks = Cg / ve;
  r.lg = 1;
  while (r.lg < 32 && r.lg < chunks) r.lg *= 2;
  r.cpl = 1;
  while ((int64_t)r.lg * r.cpl < chunks) r.cpl *= 2;
  r.ok = S == 1 && r.cpl <= 8 && r.cpl * ve <= 32;
  const int most = 256 / r.lg;  // groups (of any sample) per CTA
  r.gy = (int)((G + most - 1) / most);
  r.gpc = (int)((G + r.gy - 1) / r.gy);
  r.spc = most / r.gpc;
  // one wave of the CTAs that are resident: a thread's parameters are loaded once
  const int64_t need = (N + r.spc - 1) / r.spc, fill = ((int64_t)kGnSms * (bwd ? 2 : 4) + r.gy - 1) / r.gy;
  r.ctas = need < fill ? need : fill;
  return r;
}
// Several positions.  One pass when a sample's block of some 64 channels is small enough (64 KB in
// bf16) to be read again from L1 (2 x 225 x 96: 6.0 us forward, 7.2 backward; in two passes 7.6 and
// 10.5).  Else slices of each sample, 32 positions or more, in one wave of the resident CTAs: a
// CTA's fixed cost (joining its threads' sums) is that of some 30 rows, and a second wave starts
// late (432 backward CTAs for 296 places: 60 us, 296: 46 us, 4 x 16384 x 128 fp32).  Also tried: the
// block held in the shared memory of a cluster and read once (16 x 4096 x 320 bf16: 51 us for 34).
struct GnPlan { int64_t slices, rows, cb, gz; bool one; };
// Whole groups, about `want` channels, a multiple of the channels that a load of the full row
// could take (so that blocks do not narrow the loads) as long as the block's sums, two floats a
// channel where a thread has several chunks, stay within the 48 KB that a launch may ask for: wide
// odd groups take narrower loads instead (gn_width goes by the block too).
constexpr int64_t kGnMostBlock = 48 * 1024 / 8;
static_assert(kGnMostCg <= kGnMostBlock, "a block holds at least one group");
static int64_t gn_block(int64_t C, int64_t Cg, int64_t want) {
  int64_t step = Cg;
  for (int ve = 2; ve <= 8 && C % ve == 0; ve *= 2) {  // step is a multiple of ve / 2
    if (step % ve == 0) continue;
    if (2 * step > kGnMostBlock) break;
    step *= 2;
  }
  if (C <= want || C <= step) return C;
  return step >= want ? step : want / step * step;
}
static GnPlan gn_plan(int64_t N, int64_t S, int64_t C, int64_t G, bool bwd) {
  GnPlan r{};
  const int64_t Cg = C / G;
  r.cb = gn_block(C, Cg, 64);
  r.one = S * r.cb <= 32768 && r.cb <= 1024;
  if (!r.one) r.cb = gn_block(C, Cg, 512);
  r.gz = (C + r.cb - 1) / r.cb;
  r.rows = S;
  r.slices = 1;
  if (!r.one) {
    const int64_t ctas = kGnSms * (bwd ? kGnBwdCtas : kGnFwdCtas), want = ctas >= N * r.gz ? ctas / (N * r.gz) : 1;
    r.rows = (S + want - 1) / want;
    if (r.rows < 32) r.rows = S < 32 ? S : 32;
    r.slices = (S + r.rows - 1) / r.rows;
  }
  return r;
}
static int gn_width(int es, int64_t d);
// What a call of element size es needs in its workspace (that of a shape is the larger one of both
// types').  Forward: the slices' statistics, then the samples' mean and rstd when the caller does not
// want them.  Gradient: the row CTAs' sums, or the slices' sums, the samples' sums (where a sample
// has several slices) and the groups' means.
static size_t gn_fwd_ws(int es, int64_t N, int64_t S, int64_t C, int64_t G) {
  if (C / G > kGnMostCg || gn_row_plan(N, S, G, C / G, gn_width(es, C / G)).ok) return 0;
  const GnPlan r = gn_plan(N, S, C, G, false);
  return r.one ? 0 : (size_t)N * G * 8 * (r.slices + 1);
}
static size_t gn_bwd_ws(int es, int64_t N, int64_t S, int64_t C, int64_t G) {
  if (C / G > kGnMostCg) return (size_t)N * 2 * C * 4;
  const GnRowPlan row = gn_row_plan(N, S, G, C / G, gn_width(es, C / G), true);
  if (row.ok) return (size_t)row.ctas * 2 * C * 4;
  const GnPlan r = gn_plan(N, S, C, G, true);
  return (size_t)N * 2 * 4 * ((r.slices > 1 ? r.slices + 1 : 1) * C + (r.one ? 0 : G));
}
// Channels per load: as many as 16 bytes hold and divide d (the group's channels, or the row's).
// The layout does not enter, so that it does not change the arithmetic; whether the rows allow
// such loads does (whole).
static int gn_width(int es, int64_t d) {
  int ve = 16 / es;
  while (d % ve != 0) ve /= 2;
  return ve;
}
static int gn_whole(int es, int ve, const void* const* ptr, const int64_t* stride, int n) {
  bool ok = true;
  for (int i = 0; i < n; ++i)
    ok = ok && reinterpret_cast<uintptr_t>(ptr[i]) % (ve * es) == 0 && stride[2 * i] % ve == 0 && stride[2 * i + 1] % ve == 0;
  return ok;
}

enum GnPass { kStats, kApply, kSums, kDx };
template <typename T, int VE, bool WHOLE>
static void gn_pass(GnPass pass, const GnParams& p, const GnPlan& r, cudaStream_t s) {
  const dim3 grid((unsigned)(r.slices * p.N), (unsigned)r.gz);
  // the row lanes' values of the widest block; a narrower last one has no more of them
  const size_t values = (size_t)2 * gn_lanes((int)(r.cb / VE)) * r.cb > 2 * kGnThreads * VE
                            ? (size_t)2 * gn_lanes((int)(r.cb / VE)) * r.cb : 2 * kGnThreads * VE;
  const size_t groups = 2 * (r.cb / p.Cg), smem = (values + (r.one ? groups : 0)) * 4;
  const size_t smem_sums = (values + (r.one ? 2 * r.cb + groups : 0)) * 4;
  switch (pass) {
    case kStats:
      if (r.one) gn_stats_kernel<T, VE, WHOLE, true><<<grid, kGnThreads, smem, s>>>(p);
      else gn_stats_kernel<T, VE, WHOLE, false><<<grid, kGnThreads, smem, s>>>(p);
      break;
    case kApply: launch_dependent(gn_apply_kernel<T, VE, WHOLE>, grid, kGnThreads, 0, s, p); break;
    case kSums:
      if (r.one) gn_sums_kernel<T, VE, WHOLE, true><<<grid, kGnThreads, smem_sums, s>>>(p);
      else gn_sums_kernel<T, VE, WHOLE, false><<<grid, kGnThreads, smem_sums, s>>>(p);
      break;
    case kDx: launch_dependent(gn_dx_kernel<T, VE, WHOLE>, grid, kGnThreads, 0, s, p); break;
  }
}
template <typename T, int VE> static void gn_pass(GnPass pass, const GnParams& p, const GnPlan& r, cudaStream_t s) {
  if (VE == 1 || p.whole) gn_pass<T, VE, true>(pass, p, r, s);
  else gn_pass<T, VE, VE == 1>(pass, p, r, s);
}
template <typename T> static void gn_pass(GnPass pass, const GnParams& p, const GnPlan& r, int ve, cudaStream_t s) {
  if (ve == 1) return gn_pass<T, 1>(pass, p, r, s);
  if (ve == 2) return gn_pass<T, 2>(pass, p, r, s);
  if (ve == 4) return gn_pass<T, 4>(pass, p, r, s);
  if constexpr (sizeof(T) == 2) return gn_pass<T, 8>(pass, p, r, s);
}
static void gn_pass(GnPass pass, int dtype, const GnParams& p, const GnPlan& r, int ve, cudaStream_t s) {
  if (dtype == HDC_F32) gn_pass<float>(pass, p, r, ve, s);
  else gn_pass<__nv_bfloat16>(pass, p, r, ve, s);
}

static bool gn_off(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == HDC_F32 ? 3u : 1u)) != 0;
}

static int gn_check(const char* what, int dtype, int p_dtype, int64_t N, int64_t S, int64_t C, int64_t G, int act) {
  if ((dtype != HDC_F32 && dtype != HDC_BF16) || (p_dtype != HDC_F32 && p_dtype != HDC_BF16))
    return fail(HDC_E_DTYPE, "%s: dtype %d, parameter dtype %d", what, dtype, p_dtype);
  if (act != HDC_ACT_NONE && act != HDC_ACT_SILU) return fail(HDC_E_SHAPE, "%s: activation %d", what, act);
  if (N < 0 || S < 0 || C < 1 || G < 1 || C % G != 0 || C > 65536 || N > (int64_t(1) << 30) ||
      S > (int64_t(1) << 30) || N * G >= (int64_t(1) << 31))
    return fail(HDC_E_SHAPE, "%s: N=%lld, S=%lld, C=%lld (1..65536), G=%lld (a divisor of C), N*G < 2^31", what,
                (long long)N, (long long)S, (long long)C, (long long)G);
  return 0;
}

}  // namespace hdc

using namespace hdc;

extern "C" size_t hdc_group_norm_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G) {
  if (N < 1 || S < 1 || C < 1 || G < 1 || C % G != 0) return 0;
  const size_t a = gn_fwd_ws(2, N, S, C, G), b = gn_fwd_ws(4, N, S, C, G);
  return a > b ? a : b;
}

extern "C" int hdc_group_norm_fwd(int dtype, int p_dtype, const void* x, int64_t x_sn, int64_t x_ss, const void* weight,
                                  const void* bias, void* y, int64_t y_sn, int64_t y_ss, float* mean, float* rstd,
                                  void* workspace, size_t workspace_bytes, int64_t N, int64_t S, int64_t C, int64_t G,
                                  float eps, int act, hdc_stream_t stream) {
  if (int e = gn_check("group_norm", dtype, p_dtype, N, S, C, G, act)) return e;
  if (N == 0 || S == 0) return HDC_OK;
  if (!x || !y || (!mean != !rstd)) return fail(HDC_E_NULL, "group_norm: null pointer");
  if (gn_off(x, dtype) || gn_off(y, dtype) || gn_off(weight, p_dtype) || gn_off(bias, p_dtype) ||
      gn_off(mean, HDC_F32) || gn_off(rstd, HDC_F32) || !aligned16(workspace))
    return fail(HDC_E_ALIGN, "group_norm: a pointer is not aligned to its type");
  if (!rows_apart(N, y_sn, S, y_ss, C))
    return fail(HDC_E_SHAPE, "group_norm: y rows overlap (y_sn=%lld, y_ss=%lld)", (long long)y_sn, (long long)y_ss);
  const size_t need = hdc_group_norm_workspace_bytes(N, S, C, G);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(HDC_E_WORKSPACE, "group_norm: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  GnParams p{};
  p.x = x; p.xsn = x_sn; p.xss = x_ss; p.w = weight; p.b = bias; p.p_bf16 = p_dtype == HDC_BF16;
  p.y = y; p.ysn = y_sn; p.yss = y_ss; p.mean = mean; p.rstd = rstd; p.stats = static_cast<float2*>(workspace);
  p.N = (int)N; p.S = (int)S; p.C = (int)C; p.G = (int)G; p.Cg = (int)(C / G); p.eps = eps;
  p.silu = act == HDC_ACT_SILU;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  const int es = dtype == HDC_F32 ? 4 : 2;
  if (p.Cg > kGnMostCg) {
    if (dtype == HDC_F32) gn_any_fwd_kernel<float><<<(unsigned)(N * G), 256, 0, s>>>(p);
    else gn_any_fwd_kernel<__nv_bfloat16><<<(unsigned)(N * G), 256, 0, s>>>(p);
    return launch_status("gn_any_fwd_kernel");
  }
  const void* ptr[] = {x, y};
  const int64_t stride[] = {N > 1 ? x_sn : 0, S > 1 ? x_ss : 0, N > 1 ? y_sn : 0, S > 1 ? y_ss : 0};
  int ve = gn_width(es, p.Cg);
  const GnRowPlan row = gn_row_plan(N, S, G, p.Cg, ve);
  if (row.ok) {
    p.whole = gn_whole(es, ve, ptr, stride, 2);
    gn_rows_fwd(dtype, p, row, ve, s);
    return launch_status("gn_row_kernel");
  }
  const GnPlan plan = gn_plan(N, S, C, G, false);
  p.slices = (int)plan.slices; p.rows = (int)plan.rows; p.cb = (int)plan.cb;
  ve = gn_width(es, plan.cb | C);
  p.whole = gn_whole(es, ve, ptr, stride, 2);
  if (!p.mean && !plan.one) {
    p.mean = reinterpret_cast<float*>(p.stats + N * plan.slices * G);
    p.rstd = p.mean + N * G;
  }
  gn_pass(kStats, dtype, p, plan, ve, s);
  if (int e = launch_status("gn_stats_kernel")) return e;
  if (plan.one) return HDC_OK;
  launch_dependent(gn_join_kernel, dim3((unsigned)((N * G + 7) / 8)), 256, 0, s, p);
  if (int e = launch_status("gn_join_kernel")) return e;
  gn_pass(kApply, dtype, p, plan, ve, s);
  return launch_status("gn_apply_kernel");
}

extern "C" size_t hdc_group_norm_bwd_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G) {
  if (N < 1 || S < 1 || C < 1 || G < 1 || C % G != 0) return 0;
  const size_t a = gn_bwd_ws(2, N, S, C, G), b = gn_bwd_ws(4, N, S, C, G);
  return a > b ? a : b;
}
// the middle step's channels per CTA: whole groups, some 64 channels
static int gn_mid_block(int C, int Cg) {
  const int b = Cg >= 64 ? Cg : 64 / Cg * Cg;
  return b < C ? b : C;
}

extern "C" int hdc_group_norm_bwd(int dtype, int p_dtype, const void* dy, int64_t dy_sn, int64_t dy_ss, const void* x,
                                  int64_t x_sn, int64_t x_ss, const float* mean, const float* rstd, const void* weight,
                                  const void* bias, void* dx, int64_t dx_sn, int64_t dx_ss, void* dweight, void* dbias,
                                  void* workspace, size_t workspace_bytes, int64_t N, int64_t S, int64_t C, int64_t G,
                                  int act, hdc_stream_t stream) {
  if (int e = gn_check("group_norm_bwd", dtype, p_dtype, N, S, C, G, act)) return e;
  const bool empty = N == 0 || S == 0;
  if (!empty && (!dy || !x || !mean || !rstd || !dx)) return fail(HDC_E_NULL, "group_norm_bwd: null pointer");
  if (gn_off(dy, dtype) || gn_off(x, dtype) || gn_off(dx, dtype) || gn_off(weight, p_dtype) || gn_off(bias, p_dtype) ||
      gn_off(dweight, p_dtype) || gn_off(dbias, p_dtype) || gn_off(mean, HDC_F32) || gn_off(rstd, HDC_F32) ||
      !aligned16(workspace))
    return fail(HDC_E_ALIGN, "group_norm_bwd: a pointer is not aligned to its type");
  if (!empty && !rows_apart(N, dx_sn, S, dx_ss, C))
    return fail(HDC_E_SHAPE, "group_norm_bwd: dx rows overlap (dx_sn=%lld, dx_ss=%lld)", (long long)dx_sn,
                (long long)dx_ss);
  const size_t need = hdc_group_norm_bwd_workspace_bytes(N, S, C, G);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(HDC_E_WORKSPACE, "group_norm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  GnParams p{};
  p.x = x; p.xsn = x_sn; p.xss = x_ss; p.w = weight; p.b = bias; p.p_bf16 = p_dtype == HDC_BF16;
  p.dy = dy; p.dsn = dy_sn; p.dss = dy_ss; p.dx = dx; p.gsn = dx_sn; p.gss = dx_ss;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd); p.part = static_cast<float*>(workspace);
  p.N = (int)N; p.S = (int)S; p.C = (int)C; p.G = (int)G; p.Cg = (int)(C / G); p.silu = act == HDC_ACT_SILU;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  const int es = dtype == HDC_F32 ? 4 : 2;
  int64_t parts = 0;
  if (!empty && p.Cg > kGnMostCg) {
    if (dtype == HDC_F32) gn_any_bwd_kernel<float><<<(unsigned)(N * G), 256, 0, s>>>(p);
    else gn_any_bwd_kernel<__nv_bfloat16><<<(unsigned)(N * G), 256, 0, s>>>(p);
    if (int e = launch_status("gn_any_bwd_kernel")) return e;
    parts = N;
  } else if (!empty) {
    const void* ptr[] = {x, dy, dx};
    const int64_t stride[] = {N > 1 ? x_sn : 0,  S > 1 ? x_ss : 0,  N > 1 ? dy_sn : 0,
                              S > 1 ? dy_ss : 0, N > 1 ? dx_sn : 0, S > 1 ? dx_ss : 0};
    int ve = gn_width(es, p.Cg);
    const GnRowPlan row = gn_row_plan(N, S, G, p.Cg, ve, true);
    if (row.ok) {
      p.whole = gn_whole(es, ve, ptr, stride, 3);
      gn_rows_bwd(dtype, p, row, ve, s);
      if (int e = launch_status("gn_row_kernel")) return e;
      parts = row.ctas;
    } else {
      const GnPlan plan = gn_plan(N, S, C, G, true);
      p.slices = (int)plan.slices; p.rows = (int)plan.rows; p.cb = (int)plan.cb;
      ve = gn_width(es, plan.cb | C);
      p.whole = gn_whole(es, ve, ptr, stride, 3);
      // a single slice's sums are the sample's: the middle step writes them where it read them
      p.sums = plan.slices > 1 ? p.part + N * plan.slices * 2 * C : p.part;
      p.gmean = p.sums + N * 2 * C;
      gn_pass(kSums, dtype, p, plan, ve, s);
      if (int e = launch_status("gn_sums_kernel")) return e;
      parts = N;
      if (!plan.one) {
        // shared memory: at most 256 threads' strands of any block, or the items of a wide one (32 KB
        // for the widest group, within the 48 KB that a launch may ask for)
        const int block = gn_mid_block(p.C, p.Cg), items = 2 * block;
        static_assert(2 * kGnMostCg * 4 <= 48 * 1024, "the middle step's sums of a group");
        launch_dependent(gn_mid_kernel, dim3((unsigned)N, (unsigned)((C + block - 1) / block)), 256,
                         (size_t)(items < 256 ? 256 : items) * 4, s, p, block);
        if (int e = launch_status("gn_mid_kernel")) return e;
        gn_pass(kDx, dtype, p, plan, ve, s);
        if (int e = launch_status("gn_dx_kernel")) return e;
        p.part = p.sums;
      }
    }
  }
  if (!dweight && !dbias) return HDC_OK;
  launch_dependent(gn_param_grad_kernel, dim3((unsigned)((C + 31) / 32), 2), 1024, 0, s, p.part, parts, (int)C, dweight,
                   dbias, p.p_bf16);
  return launch_status("gn_param_grad_kernel");
}
