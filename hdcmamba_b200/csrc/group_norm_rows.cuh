// Group norm of one position per sample: kernel and launches (one direction per source file).
//
// Bound by HBM in bytes, in fact by issue slots and the two MUFU operations (2^x, 1/x) of each
// SiLU: 32768 x 16 heads of 64 bf16 forward 29 us (71% of 6550 GB/s), backward 45 us (68%); 17 and
// 26 M warp instructions, 58 to 60% of the issue slots busy.  What brought it there: loads known
// to be whole at compile time (72 -> 56 us backward), one wave of resident CTAs (87 -> 72), the
// next sample's loads in flight during this one's arithmetic (56 -> 47), pairs of fp32 (31 -> 26
// forward at 12 heads).
#pragma once
#include "group_norm.cuh"

namespace hdc {

// ---------------------------------------------------------------- one position per sample
// The lanes of a group: LG of them, CPL loads of VE channels each: channel (k LG + l) VE + i of
// the group.  Threads: (sample of the CTA, group, lane), groups from blockIdx.y * gpc.
// FULL: the lanes' loads are exactly the group.
// LG 0: known only at run time (lg).
template <int LG> __device__ __forceinline__ float group_sum(float v, int lg) {
  if constexpr (LG == 0) {
    for (int o = lg / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  } else {
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

template <typename T, int VE, bool WHOLE, int CPL, int U, bool BWD, int LG, bool FULL>
__global__ void __launch_bounds__(256) gn_row_kernel(const __grid_constant__ GnParams p, int gpc, int spc, int lanes) {
  const int lg = LG ? LG : lanes;
  const int l = threadIdx.x & (lg - 1), gi = threadIdx.x / lg % gpc, sr = threadIdx.x / lg / gpc;
  const int g = blockIdx.y * gpc + gi;
  const bool live = g < p.G && sr < spc;
  const int gc = live ? g : 0, c0 = gc * p.Cg;
  constexpr int M = VE * CPL;
  int ch[CPL];
  bool in[CPL];
  Fv<VE> w[CPL], b[CPL], dw[BWD ? CPL : 1], db[BWD ? CPL : 1];
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int c = (k * lg + l) * VE;
    in[k] = FULL || c < p.Cg;
    ch[k] = c0 + (in[k] ? c : 0);
    w[k] = gn_params<VE>(p.w, p.p_bf16, ch[k], 1.f);
    b[k] = gn_params<VE>(p.b, p.p_bf16, ch[k], 0.f);
    if constexpr (BWD) dw[k] = db[k] = all<VE>(0.f);
  }
  const float inv = 1.f / (float)p.Cg;
  if constexpr (BWD) let_next_start();

  // The thread's samples: first, first + step, ...  All threads of the CTA take the same number of
  // turns (the shuffles want whole warps); a turn past the last sample, or a thread without a
  // group, reads the thread's first sample (or sample 0) again and stores nothing.
  const int64_t step = (int64_t)gridDim.x * spc, cta0 = (int64_t)blockIdx.x * spc;
  const bool any = live && cta0 + sr < p.N;
  const int64_t first = any ? cta0 + sr : 0;
  const int turns = (int)((p.N - cta0 + step - 1) / step);                          // of the CTA
  const int whole_turns = any && first + (turns - 1) * step < p.N ? turns : any ? turns - 1 : 0;  // of the thread
  const T* xp = static_cast<const T*>(p.x) + first * p.xsn;
  const T* dp = static_cast<const T*>(p.dy) + first * p.dsn;
  T* op = (BWD ? static_cast<T*>(p.dx) : static_cast<T*>(p.y)) + first * (BWD ? p.gsn : p.ysn);
  float* mp = p.mean ? p.mean + first * p.G + gc : nullptr;
  float* rp = p.mean ? p.rstd + first * p.G + gc : nullptr;
  const int64_t xs = step * p.xsn, ds = step * p.dsn, os = step * (BWD ? p.gsn : p.ysn), gs = step * p.G;
  const bool stats = !BWD && l == 0 && mp;

  struct Turn {
    Raw<T, VE> x[CPL], dy[BWD ? CPL : 1];
    float mu, rs;
  };
  auto load = [&](int i) {
    const int64_t at = i < whole_turns ? i : 0;
    Turn t;
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      t.x[k] = ld_raw<T, VE, WHOLE, !BWD>(xp + at * xs + ch[k]);
      if constexpr (BWD) t.dy[k] = ld_raw<T, VE, WHOLE, !BWD>(dp + at * ds + ch[k]);
    }
    if constexpr (BWD) {
      t.mu = __ldg(mp + at * gs);
      t.rs = __ldg(rp + at * gs);
    }
    return t;
  };
  // the loads of the next U turns are in flight during U turns
  Turn next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = load(u);
  for (int i = 0; i < turns; i += U) {
    Turn now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = next[u];
    if (i + U < turns) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = load(i + U + u);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = i + u < whole_turns;
      Fv<VE> x[CPL];
      if constexpr (!BWD) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          x[k] = unpack<T, VE>(now[u].x[k]);
          s += in[k] ? sum_of(x[k]) : 0.f;
        }
        const float mean = over(group_sum<LG>(s, lg), (float)p.Cg, inv);
        s = 0.f;
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          x[k] = x[k] + all<VE>(-mean);
          s += in[k] ? sum_of(x[k] * x[k]) : 0.f;
        }
        const float rstd = gn_rstd(group_sum<LG>(s, lg), inv, p.eps);
        if (ok) {
#pragma unroll
          for (int k = 0; k < CPL; ++k)
            if (in[k])
              st_vec<T, VE, WHOLE>(op + (i + u) * os + ch[k], gn_act<T>(fma(x[k] * all<VE>(rstd), w[k], b[k]), p.silu));
          if (stats) {
            mp[(i + u) * gs] = mean;
            rp[(i + u) * gs] = rstd;
          }
        }
      } else {
        Fv<VE> e[CPL];
        float se = 0.f, sx = 0.f;
#pragma unroll
        for (int k = 0; k < CPL; ++k) {
          x[k] = (unpack<T, VE>(now[u].x[k]) + all<VE>(-now[u].mu)) * all<VE>(now[u].rs);
          const Fv<VE> dz = gn_dact<T>(unpack<T, VE>(now[u].dy[k]), fma(x[k], w[k], b[k]), p.silu);
          e[k] = dz * w[k];
          if (ok && in[k]) {
            dw[k] = fma(dz, x[k], dw[k]);
            db[k] = db[k] + dz;
            se += sum_of(e[k]);
            sx += sum_of(e[k] * x[k]);
          }
        }
        se = group_sum<LG>(se, lg) * inv;
        sx = group_sum<LG>(sx, lg) * inv;
        if (ok) {
#pragma unroll
          for (int k = 0; k < CPL; ++k)
            if (in[k])
              st_vec<T, VE, WHOLE>(op + (i + u) * os + ch[k],
                            fma(x[k], all<VE>(-sx), e[k] + all<VE>(-se)) * all<VE>(now[u].rs));
        }
      }
    }
  }
  if constexpr (BWD) {  // the CTA's sums over its samples, in their order
    extern __shared__ float sh[];  // [spc][M][gpc * lg]
    const int per = gpc * lg, q = threadIdx.x % per;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      if (sr < spc) {
#pragma unroll
        for (int i = 0; i < M; ++i) sh[((size_t)sr * M + i) * per + q] = (which ? db[i / VE] : dw[i / VE]).v[i % VE];
      }
      __syncthreads();
      if (sr == 0 && live) {
#pragma unroll
        for (int k = 0; k < CPL; ++k)
          if (in[k])
#pragma unroll
            for (int i = 0; i < VE; ++i) {
              float v = 0.f;
              for (int r = 0; r < spc; ++r) v += sh[((size_t)r * M + k * VE + i) * per + q];
              p.part[((int64_t)blockIdx.x * 2 + which) * p.C + ch[k] + i] = v;
            }
      }
    }
  }
}

template <typename T, int VE, bool WHOLE, int CPL, bool BWD, int LG, bool FULL>
static void gn_row_launch(const GnParams& p, const GnRowPlan& r, cudaStream_t s) {
  constexpr int M = VE * CPL, U = M <= 8 ? 2 : 1;
  const int threads = (r.gpc * r.lg * r.spc + 31) / 32 * 32;
  const size_t smem = BWD ? (size_t)r.spc * r.gpc * r.lg * M * 4 : 0;
  gn_row_kernel<T, VE, WHOLE, CPL, U, BWD, LG, FULL>
      <<<dim3((unsigned)r.ctas, (unsigned)r.gy), threads, smem, s>>>(p, r.gpc, r.spc, r.lg);
}
// The widest loads of groups that the lanes cover exactly: the number of lanes known at compile
// time, no bounds within a group.  All others by the general form (the same arithmetic).
template <typename T, int VE, int CPL, bool BWD>
static bool gn_row_exact(const GnParams& p, const GnRowPlan& r, cudaStream_t s) {
  if (VE * (int)sizeof(T) != 16 || !p.whole || r.lg * CPL * VE != p.Cg) return false;
  if constexpr (VE * (int)sizeof(T) == 16) {
    if constexpr (CPL == 1) {
      switch (r.lg) {
        case 1: gn_row_launch<T, VE, true, 1, BWD, 1, true>(p, r, s); return true;
        case 2: gn_row_launch<T, VE, true, 1, BWD, 2, true>(p, r, s); return true;
        case 4: gn_row_launch<T, VE, true, 1, BWD, 4, true>(p, r, s); return true;
        case 8: gn_row_launch<T, VE, true, 1, BWD, 8, true>(p, r, s); return true;
        case 16: gn_row_launch<T, VE, true, 1, BWD, 16, true>(p, r, s); return true;
      }
    }
    gn_row_launch<T, VE, true, CPL, BWD, 32, true>(p, r, s);  // more loads than one, so all 32 lanes
  }
  return true;
}
template <typename T, int VE, int CPL, bool BWD>
static void gn_row_loads(const GnParams& p, const GnRowPlan& r, cudaStream_t s) {
  if (gn_row_exact<T, VE, CPL, BWD>(p, r, s)) return;
  if (VE == 1 || p.whole) gn_row_launch<T, VE, true, CPL, BWD, 0, false>(p, r, s);
  else gn_row_launch<T, VE, VE == 1, CPL, BWD, 0, false>(p, r, s);
}
template <typename T, int VE, bool BWD> static void gn_row_width(const GnParams& p, const GnRowPlan& r, cudaStream_t s) {
  if (r.cpl == 1) return gn_row_loads<T, VE, 1, BWD>(p, r, s);
  if (r.cpl == 2) return gn_row_loads<T, VE, 2, BWD>(p, r, s);
  if (r.cpl == 4) return gn_row_loads<T, VE, 4, BWD>(p, r, s);
  if constexpr (VE <= 4) return gn_row_loads<T, VE, 8, BWD>(p, r, s);
}
template <typename T, bool BWD> static void gn_rows(const GnParams& p, const GnRowPlan& r, int ve, cudaStream_t s) {
  if (ve == 1) return gn_row_width<T, 1, BWD>(p, r, s);
  if (ve == 2) return gn_row_width<T, 2, BWD>(p, r, s);
  if (ve == 4) return gn_row_width<T, 4, BWD>(p, r, s);
  if constexpr (sizeof(T) == 2) return gn_row_width<T, 8, BWD>(p, r, s);
}

}  // namespace hdc
