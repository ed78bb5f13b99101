// Short vectors of fp32 values, computed as pairs (fma.rn.f32x2 and friends: two fp32 operations
// per issued instruction), and the hardware's 2^x and 1/x.
#pragma once
#include "common.cuh"

namespace hdc {

template <int V> struct Fv { float v[V]; };

__device__ __forceinline__ uint64_t pair_bits(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void bits_pair(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
template <int V> __device__ __forceinline__ Fv<V> fma(const Fv<V>& a, const Fv<V>& b, const Fv<V>& c) {
  Fv<V> o;
  if constexpr (V == 1) {
    o.v[0] = fmaf(a.v[0], b.v[0], c.v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      uint64_t r;
      asm("fma.rn.f32x2 %0, %1, %2, %3;"
          : "=l"(r)
          : "l"(pair_bits(a.v[i], a.v[i + 1])), "l"(pair_bits(b.v[i], b.v[i + 1])), "l"(pair_bits(c.v[i], c.v[i + 1])));
      bits_pair(r, o.v[i], o.v[i + 1]);
    }
  }
  return o;
}
template <int V> __device__ __forceinline__ Fv<V> operator*(const Fv<V>& a, const Fv<V>& b) {
  Fv<V> o;
  if constexpr (V == 1) {
    o.v[0] = a.v[0] * b.v[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      uint64_t r;
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a.v[i], a.v[i + 1])), "l"(pair_bits(b.v[i], b.v[i + 1])));
      bits_pair(r, o.v[i], o.v[i + 1]);
    }
  }
  return o;
}
template <int V> __device__ __forceinline__ Fv<V> operator+(const Fv<V>& a, const Fv<V>& b) {
  Fv<V> o;
  if constexpr (V == 1) {
    o.v[0] = a.v[0] + b.v[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      uint64_t r;
      asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a.v[i], a.v[i + 1])), "l"(pair_bits(b.v[i], b.v[i + 1])));
      bits_pair(r, o.v[i], o.v[i + 1]);
    }
  }
  return o;
}
template <int V> __device__ __forceinline__ Fv<V> all(float x) {
  Fv<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = x;
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// After this, memory written by the kernels before this one on the stream may be read, when it
// was launched as a programmatic dependent (otherwise it returns at once).
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The dependent launch may start (its CTAs then wait as above).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;"); }

// Launch k as a programmatic dependent of the kernel before it on the stream.
template <typename... P, typename... A>
inline void launch_dependent(void (*k)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, k, P(args)...);
}

}  // namespace hdc
