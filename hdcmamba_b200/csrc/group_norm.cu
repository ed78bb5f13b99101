// Group norm with an activation, channels last, sm_100a: forward and gradient.
//
// x [N, S, C], G groups of Cg = C/G channels; statistics of (n, g) over its S*Cg values:
//   xh = (x - mean) rstd,  z = xh w_c + b_c,  y = act(z)      (act: none or z sigmoid(z))
//   dz = dy act'(z),  dw_c = sum_{n,s} dz xh,  db_c = sum_{n,s} dz,  e = dz w_c
//   dx = rstd (e - mean_g(e) - xh mean_g(e xh))
// S = 1 is the Block's norm of each head and token (hdcmamba/model.py:285-292).
// Statistics and sums are fp32; y, dx, dw, db are rounded once to their types.
//
// Schedule: one CTA per (n, g).
#include "common.cuh"

namespace hdc {

struct GnParams {
  const void* x; int64_t xsn, xss;
  const void* w; const void* b; int p_bf16;
  void* y; int64_t ysn, yss;
  float* mean; float* rstd;
  const void* dy; int64_t dsn, dss;
  void* dx; int64_t gsn, gss;
  float* part;  // [N, 2, C] sums of dz xh and dz
  int N, S, C, G, Cg;
  float eps; int silu;
};

__device__ __forceinline__ float gn_param(const void* p, int bf16, int i, float none) {
  if (!p) return none;
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

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
__global__ void __launch_bounds__(256) gn_fwd_kernel(GnParams p) {
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
  const float rstd = 1.f / sqrtf(block_sum(s) / (float)M + p.eps);
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
__global__ void __launch_bounds__(256) gn_bwd_kernel(GnParams p) {
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

// dw[c], db[c]: sums of the parts in their order (blockIdx.y: 0 dw, 1 db)
__global__ void gn_param_grad_kernel(const float* part, int parts, int C, void* dw, void* db, int bf16) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= C) return;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0.f;
  for (int k = 0; k < parts; ++k) s += part[((int64_t)k * 2 + blockIdx.y) * C + c];
  if (bf16) static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(s);
  else static_cast<float*>(out)[c] = s;
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

extern "C" size_t hdc_group_norm_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G) { return 0; }

extern "C" int hdc_group_norm_fwd(int dtype, int p_dtype, const void* x, int64_t x_sn, int64_t x_ss, const void* weight,
                                  const void* bias, void* y, int64_t y_sn, int64_t y_ss, float* mean, float* rstd,
                                  void* workspace, size_t workspace_bytes, int64_t N, int64_t S, int64_t C, int64_t G,
                                  float eps, int act, hdc_stream_t stream) {
  if (int e = gn_check("group_norm", dtype, p_dtype, N, S, C, G, act)) return e;
  if (N == 0 || S == 0) return HDC_OK;
  if (!x || !y || (!mean != !rstd)) return fail(HDC_E_NULL, "group_norm: null pointer");
  if (gn_off(x, dtype) || gn_off(y, dtype) || gn_off(weight, p_dtype) || gn_off(bias, p_dtype) ||
      gn_off(mean, HDC_F32) || gn_off(rstd, HDC_F32))
    return fail(HDC_E_ALIGN, "group_norm: a pointer is not aligned to its type");
  if (workspace_bytes < hdc_group_norm_workspace_bytes(N, S, C, G))
    return fail(HDC_E_WORKSPACE, "group_norm: workspace of %zu bytes is too small", workspace_bytes);
  GnParams p{};
  p.x = x; p.xsn = x_sn; p.xss = x_ss; p.w = weight; p.b = bias; p.p_bf16 = p_dtype == HDC_BF16;
  p.y = y; p.ysn = y_sn; p.yss = y_ss; p.mean = mean; p.rstd = rstd;
  p.N = (int)N; p.S = (int)S; p.C = (int)C; p.G = (int)G; p.Cg = (int)(C / G); p.eps = eps;
  p.silu = act == HDC_ACT_SILU;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == HDC_F32) gn_fwd_kernel<float><<<(unsigned)(N * G), 256, 0, s>>>(p);
  else gn_fwd_kernel<__nv_bfloat16><<<(unsigned)(N * G), 256, 0, s>>>(p);
  return launch_status("gn_fwd_kernel");
}

extern "C" size_t hdc_group_norm_bwd_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G) {
  return N > 0 && S > 0 && C > 0 ? (size_t)N * 2 * C * 4 : 0;
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
      gn_off(workspace, HDC_F32))
    return fail(HDC_E_ALIGN, "group_norm_bwd: a pointer is not aligned to its type");
  const size_t need = hdc_group_norm_bwd_workspace_bytes(N, S, C, G);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(HDC_E_WORKSPACE, "group_norm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  GnParams p{};
  p.x = x; p.xsn = x_sn; p.xss = x_ss; p.w = weight; p.b = bias; p.p_bf16 = p_dtype == HDC_BF16;
  p.dy = dy; p.dsn = dy_sn; p.dss = dy_ss; p.dx = dx; p.gsn = dx_sn; p.gss = dx_ss;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd); p.part = static_cast<float*>(workspace);
  p.N = (int)N; p.S = (int)S; p.C = (int)C; p.G = (int)G; p.Cg = (int)(C / G); p.silu = act == HDC_ACT_SILU;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  if (!empty) {
    if (dtype == HDC_F32) gn_bwd_kernel<float><<<(unsigned)(N * G), 256, 0, s>>>(p);
    else gn_bwd_kernel<__nv_bfloat16><<<(unsigned)(N * G), 256, 0, s>>>(p);
    if (int e = launch_status("gn_bwd_kernel")) return e;
  }
  if (!dweight && !dbias) return HDC_OK;
  gn_param_grad_kernel<<<dim3((unsigned)((C + 127) / 128), 2), 128, 0, s>>>(p.part, empty ? 0 : (int)N, (int)C,
                                                                           dweight, dbias, p.p_bf16);
  return launch_status("gn_param_grad_kernel");
}
