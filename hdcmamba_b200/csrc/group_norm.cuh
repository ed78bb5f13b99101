// Group norm with an activation: parameters, loads and arithmetic shared by its kernels.
#pragma once
#include "vec.cuh"

namespace hdc {

struct GnParams {
  const void* x; int64_t xsn, xss;
  const void* w; const void* b; int p_bf16;
  void* y; int64_t ysn, yss;
  float* mean; float* rstd;
  const void* dy; int64_t dsn, dss;
  void* dx; int64_t gsn, gss;
  float* part;     // gradient: sums of dz xh and of dz per channel, [part][2][C]
  float2* stats;   // two passes: (mean, M2) of each slice, [N][slices][G]
  float* sums;     // two passes, gradient: part over the slices, [N][2][C]
  float* gmean;    // and the groups' means of e xh and of e, [N][2][G]
  int N, S, C, G, Cg;
  float eps; int silu;
  int slices, rows;  // two passes: slices per sample, positions per slice
  int cb;            // two passes: channels per CTA (whole groups, or all)
  int whole;         // the rows allow whole loads (else one by one, with the same arithmetic)
};

__device__ __forceinline__ float gn_param(const void* p, int bf16, int i, float none) {
  if (!p) return none;
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

// VE neighbouring values as loaded, at once or (rows that do not allow it) one by one.  RO: nothing
// writes them while the kernel runs (the gradient's dx may be x or dy itself, so kernels that write
// dx load both the ordinary way).
template <typename T, int VE> struct Raw { static constexpr int kW = VE * (int)sizeof(T) >= 4 ? VE * (int)sizeof(T) / 4 : 1; uint32_t w[kW]; };
template <typename T, int VE, bool WHOLE, bool RO> __device__ __forceinline__ Raw<T, VE> ld_raw(const T* p) {
  Raw<T, VE> r;
  constexpr int bytes = VE * (int)sizeof(T);
  if constexpr (VE > 1 && !WHOLE) {
#pragma unroll
    for (int i = 0; i < Raw<T, VE>::kW; ++i) {
      if constexpr (sizeof(T) == 4) {
        r.w[i] = __float_as_uint(p[i]);
      } else {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p) + 2 * i;
        r.w[i] = q[0] | (uint32_t)q[VE > 1 ? 1 : 0] << 16;
      }
    }
    return r;
  }
  if constexpr (bytes == 16) {
    uint4 q;
    if constexpr (RO) q = ldg16(p);
    else asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p) : "memory");
    r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
  } else if constexpr (bytes == 8) {
    const uint2* at = reinterpret_cast<const uint2*>(p);
    const uint2 q = RO ? __ldg(at) : *at;
    r.w[0] = q.x; r.w[1] = q.y;
  } else if constexpr (bytes == 4) {
    const uint32_t* at = reinterpret_cast<const uint32_t*>(p);
    r.w[0] = RO ? __ldg(at) : *at;
  } else {
    const unsigned short* at = reinterpret_cast<const unsigned short*>(p);
    r.w[0] = RO ? __ldg(at) : *at;
  }
  return r;
}
template <typename T, int VE> __device__ __forceinline__ Fv<VE> unpack(const Raw<T, VE>& r) {
  Fv<VE> f;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    if constexpr (sizeof(T) == 4) f.v[i] = __uint_as_float(r.w[i]);
    else f.v[i] = __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
  }
  return f;
}
template <typename T, int VE, bool WHOLE> __device__ __forceinline__ void st_vec(T* p, const Fv<VE>& f) {
  constexpr int bytes = VE * (int)sizeof(T);
  if constexpr (VE > 1 && !WHOLE) {
#pragma unroll
    for (int i = 0; i < VE; ++i) p[i] = from_f<T>(f.v[i]);
    return;
  }
  if constexpr (bytes == 2) {
    *p = from_f<T>(f.v[0]);
  } else {
    uint32_t w[bytes / 4];
#pragma unroll
    for (int i = 0; i < bytes / 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(f.v[i]);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.v[2 * i], f.v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (bytes == 16) stg16(p, make_uint4(w[0], w[1], w[2], w[3]));
    else if constexpr (bytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// sigmoid: hardware 2^x and reciprocal for bf16 tensors (a few 2^-23 off), the library's for fp32
template <typename T, int V> __device__ __forceinline__ Fv<V> gn_sigmoid(const Fv<V>& z) {
  Fv<V> q;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = 1.f / (1.f + expf(-z.v[i]));
  } else {
    q = z * all<V>(-1.4426950408889634f);
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = ex2(q.v[i]);
    q = q + all<V>(1.f);
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = rcp(q.v[i]);
  }
  return q;
}
template <typename T, int V> __device__ __forceinline__ Fv<V> gn_act(const Fv<V>& z, int silu) {
  return silu ? z * gn_sigmoid<T>(z) : z;
}
// dz from dy
template <typename T, int V> __device__ __forceinline__ Fv<V> gn_dact(const Fv<V>& dy, const Fv<V>& z, int silu) {
  if (!silu) return dy;
  const Fv<V> q = gn_sigmoid<T>(z);
  return dy * (q * fma(z, fma(q, all<V>(-1.f), all<V>(1.f)), all<V>(1.f)));
}
template <int V> __device__ __forceinline__ float sum_of(const Fv<V>& f) {
  if constexpr (V >= 4) {  // halves added as pairs
    Fv<V / 2> a, b;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      a.v[i] = f.v[i];
      b.v[i] = f.v[V / 2 + i];
    }
    return sum_of(a + b);
  } else if constexpr (V == 2) {
    return f.v[0] + f.v[1];
  } else {
    return f.v[0];
  }
}
template <int V> __device__ __forceinline__ Fv<V> gn_params(const void* p, int bf16, int c, float none) {
  Fv<V> f;
#pragma unroll
  for (int i = 0; i < V; ++i) f.v[i] = gn_param(p, bf16, c + i, none);
  return f;
}
// s / n given inv = 1 / n: one correction makes up for inv's rounding (a constant group's mean is
// its value)
__device__ __forceinline__ float over(float s, float n, float inv) {
  const float m = s * inv;
  return fmaf(fmaf(-m, n, s), inv, m);
}
__device__ __forceinline__ float gn_rstd(float M2, float inv, float eps) { return rsqrtf(fmaf(M2, inv, eps)); }

// Schedule of one position per sample (group_norm_rows.cuh)
// One position: loads of ve channels, LG lanes and CPL loads per group.
struct GnRowPlan { bool ok; int lg, cpl, gpc, spc, gy; int64_t ctas; };
void gn_rows_fwd(int dtype, const GnParams& p, const GnRowPlan& r, int ve, cudaStream_t s);
void gn_rows_bwd(int dtype, const GnParams& p, const GnRowPlan& r, int ve, cudaStream_t s);

}  // namespace hdc
