// Decayed linear attention on CUDA cores: products of fp32 tiles in shared memory.
#include <atomic>

#include "decay_attn.cuh"
#include "vec.cuh"

namespace hdc {

constexpr int kPitchP = kAttnChunk + 4;

template <int DP>
__device__ __forceinline__ void load_rows(float* s, const AttnView& v, int64_t at, int t0, int n, int D) {
  for (int i = threadIdx.x; i < kAttnChunk * DP; i += 256) {
    const int r = i / DP, c = i % DP;
    float x = 0.f;
    if (r < n && c < D) x = static_cast<const float*>(v.p)[at + (int64_t)(t0 + r) * v.st + c];
    s[r * (DP + 4) + c] = x;
  }
}

template <int DP>
__device__ __forceinline__ float4 at4(const float* s, int r, int c) {
  return *reinterpret_cast<const float4*>(s + r * (DP + 4) + c);
}

// 256 threads as 16 x 16: each has 4 x 4 values of a product's 64 x 64 (DP = 128: of each quarter).
template <int DP, bool OUT>
__global__ void __launch_bounds__(256) attn_simt_kernel(AttnParams p) {
  extern __shared__ float4 smem4[];
  constexpr int NT = DP / 64;
  float* Y = reinterpret_cast<float*>(smem4);
  float* Z = Y + kAttnChunk * (DP + 4);
  float* R = Z + kAttnChunk * (DP + 4);
  float* X = R + DP * (DP + 4);
  float* P = X + kAttnChunk * (DP + 4);
  __shared__ float pw[kAttnChunk + 1];
  const AttnPass& a = p.pass[blockIdx.z];
  const int D = p.D, DR = (D + 3) & ~3;
  const int64_t bh = blockIdx.x / p.nseg;
  const int seg = blockIdx.x % p.nseg;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int begin = seg * p.seg, end = min(p.L, begin + p.seg);
  const int64_t ax = b * a.x.sb + h * a.x.sh, ay = b * a.y.sb + h * a.y.sh, az = b * a.z.sb + h * a.z.sh;
  float* state = a.states + (bh * p.nseg + seg) * D * D;
  let_next_start();
  for (int i = threadIdx.x; i <= kAttnChunk; i += 256) pw[i] = decay_pow(p.g[h], i);
  if (OUT) wait_for_previous();  // the states come from the kernel before this one
  for (int i = threadIdx.x; i < DP * DP; i += 256) {
    const int r = i / DP, c = i % DP;
    float x = 0.f;
    if (OUT && r < D && c < D) x = a.transposed ? state[c * D + r] : state[r * D + c];
    R[r * (DP + 4) + c] = x;
  }
  const int chunks = (end - begin + kAttnChunk - 1) / kAttnChunk;
  for (int q = 0; q < chunks; ++q) {
    const int t0 = begin + (a.backwards ? chunks - 1 - q : q) * kAttnChunk, n = min(kAttnChunk, end - t0);
    load_rows<DP>(Y, a.y, ay, t0, n, D);
    load_rows<DP>(Z, a.z, az, t0, n, D);
    if (OUT) load_rows<DP>(X, a.x, ax, t0, n, D);
    __syncthreads();
    if (OUT) {
      float s[4][4] = {};
      for (int d = 0; d < DR; d += 4) {
        float4 u[4], w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { u[i] = at4<DP>(X, ty * 4 + i, d); w[i] = at4<DP>(Y, tx + 16 * i, d); }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            s[i][j] = fmaf(u[i].w, w[j].w, fmaf(u[i].z, w[j].z, fmaf(u[i].y, w[j].y, fmaf(u[i].x, w[j].x, s[i][j]))));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = ty * 4 + i, c = tx + 16 * j, apart = a.backwards ? c - r : r - c;
          P[r * kPitchP + c] = apart >= 0 ? a.sa * pw[apart] * s[i][j] : 0.f;
        }
      __syncthreads();
      for (int m = 0; m < NT; ++m) {
        float o[4][4] = {};
        const int c0 = tx * 4 + 64 * m;
        for (int d = 0; d < DR; d += 4) {
          float4 u[4], w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) { u[i] = at4<DP>(X, ty * 4 + i, d); w[i] = at4<DP>(R, d + i, c0); }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float uu[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              o[i][0] = fmaf(uu[k], w[k].x, o[i][0]); o[i][1] = fmaf(uu[k], w[k].y, o[i][1]);
              o[i][2] = fmaf(uu[k], w[k].z, o[i][2]); o[i][3] = fmaf(uu[k], w[k].w, o[i][3]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = ty * 4 + i, e = a.backwards ? n - 1 - r : r + 1;
          const float f = e >= 0 ? a.si * pw[e] : 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][j] *= f;
        }
        for (int d = 0; d < kAttnChunk; d += 4) {
          float4 u[4], w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[i] = *reinterpret_cast<const float4*>(P + (ty * 4 + i) * kPitchP + d);
            w[i] = at4<DP>(Z, d + i, c0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float uu[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              o[i][0] = fmaf(uu[k], w[k].x, o[i][0]); o[i][1] = fmaf(uu[k], w[k].y, o[i][1]);
              o[i][2] = fmaf(uu[k], w[k].z, o[i][2]); o[i][3] = fmaf(uu[k], w[k].w, o[i][3]);
            }
          }
        }
        float* out = static_cast<float*>(const_cast<void*>(a.out.p)) + b * a.out.sb + h * a.out.sh;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (ty * 4 + i < n && c0 + j < D) out[(int64_t)(t0 + ty * 4 + i) * a.out.st + c0 + j] = o[i][j];
      }
      __syncthreads();
    }
    for (int mr = 0; mr < NT; ++mr)
      for (int mc = 0; mc < NT; ++mc) {
        const int r0 = ty * 4 + 64 * mr, c0 = tx * 4 + 64 * mc;
        float4 s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[i] = at4<DP>(R, r0 + i, c0);
          s[i].x *= pw[n]; s[i].y *= pw[n]; s[i].z *= pw[n]; s[i].w *= pw[n];
        }
        for (int t = 0; t < n; ++t) {
          const float w = a.su * pw[a.backwards ? t + 1 : n - 1 - t];
          const float4 u = at4<DP>(Y, t, r0), v = at4<DP>(Z, t, c0);
          const float uu[4] = {u.x * w, u.y * w, u.z * w, u.w * w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[i].x = fmaf(uu[i], v.x, s[i].x); s[i].y = fmaf(uu[i], v.y, s[i].y);
            s[i].z = fmaf(uu[i], v.z, s[i].z); s[i].w = fmaf(uu[i], v.w, s[i].w);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(R + (r0 + i) * (DP + 4) + c0) = s[i];
      }
    __syncthreads();
  }
  if (!OUT)
    for (int i = threadIdx.x; i < D * D; i += 256) state[i] = R[i / D * (DP + 4) + i % D];
}

template <int DP, bool OUT>
static int attn_launch(const AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  constexpr int smem = 4 * (kAttnChunk * (DP + 4) * (OUT ? 3 : 2) + DP * (DP + 4) + (OUT ? kAttnChunk * kPitchP : 0));
  static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is set
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    cudaFuncSetAttribute(attn_simt_kernel<DP, OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const dim3 grid((unsigned)(bh * p.nseg), 1, passes);
  if (OUT) launch_dependent(attn_simt_kernel<DP, OUT>, grid, 256, smem, s, p);
  else attn_simt_kernel<DP, OUT><<<grid, 256, smem, s>>>(p);
  return launch_status(OUT ? "attn_simt_kernel" : "attn_simt_kernel (sums)");
}

int attn_sums_f32(AttnParams& p, int64_t bh, cudaStream_t s) {
  return p.D <= 64 ? attn_launch<64, false>(p, bh, 1, s) : attn_launch<128, false>(p, bh, 1, s);
}
int attn_out_f32(AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  return p.D <= 64 ? attn_launch<64, true>(p, bh, passes, s) : attn_launch<128, true>(p, bh, passes, s);
}

}  // namespace hdc
