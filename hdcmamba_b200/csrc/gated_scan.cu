// Gated linear recurrence, sm_100a: forward, gradient and single-token step.
//
// Per batch b and channel j < ds, from projs columns dt | x | b (the Block's SSM gates,
// hdcmamba/model.py:189-193, without the reference's chunk rounding):
//   d_t = softplus20(dt_t), A = -exp(A_log), a_t = exp(d_t A), u_t = d_t b_t x_t
//   h_t = a_t h_{t-1} + u_t   (h_{-1} = h0 or 0; a reset at t drops h_{t-1}),  y_t = h_t
// Gradient, with g_t = dL/dh_t in total and c_t = a_t g_t what step t hands to step t-1:
//   g_t = dy_t + c_{t+1}  (c_L = dh_last),   s_t = g_t a_t h_{t-1} = dL/d(log a_t)
//   ddt = (s A + g b x) sigmoid(dt),  dx = g d b,  db = g d x,  dA_log = sum s d A,  dh0 = c_0
// (c_t = s_t = 0 where t is a reset.)  All arithmetic is in fp32; only y and dprojs are
// rounded, once, to the activation type.
//
// Schedule: one thread per (batch, channel) walks the sequence.
#include "common.cuh"

namespace hdc {

constexpr int kStateRows = 128;  // rows per saved state

struct ScanParams {
  const void* projs; int64_t psb, pst;
  const void* A_log; int a_bf16;
  const float* h0; const uint8_t* reset;
  void* y; int64_t ysb, yst;
  float* h_last; float* states;
  // backward
  const void* dy; int64_t dsb, dst;
  const float* dh_last;
  void* dprojs; int64_t gsb, gst;
  float* dA_part; float* dh0; float* hbuf;
  int B, L, ds, NT;
};

__device__ __forceinline__ float ld_param(const void* p, int bf16, int i) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

// softplus with the Block's threshold (hdcmamba/model.py:192), exact for small exp(x) too
__device__ __forceinline__ float softplus_acc(float x) { return x > 20.0f ? x : log1pf(expf(x)); }

template <typename T>
__global__ void __launch_bounds__(128) gated_scan_fwd_kernel(ScanParams p) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)p.B * p.ds) return;
  const int b = (int)(i / p.ds), j = (int)(i - (int64_t)b * p.ds);
  const float A = -expf(ld_param(p.A_log, p.a_bf16, j));
  const T* in = static_cast<const T*>(p.projs) + b * p.psb + j;
  T* y = static_cast<T*>(p.y) + b * p.ysb + j;
  const uint8_t* rs = p.reset ? p.reset + (int64_t)b * p.L : nullptr;
  float h = p.h0 ? p.h0[i] : 0.f;
  for (int t = 0; t < p.L; ++t) {
    if (p.states && t % kStateRows == 0) p.states[((int64_t)b * p.NT + t / kStateRows) * p.ds + j] = h;
    const T* r = in + t * p.pst;
    const float d = softplus_acc(to_f(r[0]));
    const float u = d * to_f(r[2 * p.ds]) * to_f(r[p.ds]);
    h = (rs && rs[t]) ? u : fmaf(expf(d * A), h, u);
    y[t * p.yst] = from_f<T>(h);
  }
  if (p.h_last) p.h_last[i] = h;
}

template <typename T>
__global__ void __launch_bounds__(128) gated_scan_bwd_kernel(ScanParams p) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (int64_t)p.B * p.ds) return;
  const int b = (int)(i / p.ds), j = (int)(i - (int64_t)b * p.ds);
  const float A = -expf(ld_param(p.A_log, p.a_bf16, j));
  const T* in = static_cast<const T*>(p.projs) + b * p.psb + j;
  const T* dy = static_cast<const T*>(p.dy) + b * p.dsb + j;
  T* out = static_cast<T*>(p.dprojs) + b * p.gsb + j;
  const uint8_t* rs = p.reset ? p.reset + (int64_t)b * p.L : nullptr;
  float* hb = p.hbuf + (int64_t)b * p.L * p.ds + j;
  float h = 0.f;
  for (int t = 0; t < p.L; ++t) {
    if (t % kStateRows == 0) h = p.states[((int64_t)b * p.NT + t / kStateRows) * p.ds + j];
    hb[(int64_t)t * p.ds] = h;
    const T* r = in + t * p.pst;
    const float d = softplus_acc(to_f(r[0]));
    const float u = d * to_f(r[2 * p.ds]) * to_f(r[p.ds]);
    h = (rs && rs[t]) ? u : fmaf(expf(d * A), h, u);
  }
  float c = p.dh_last ? p.dh_last[i] : 0.f;
  float dA = 0.f;
  for (int t = p.L - 1; t >= 0; --t) {
    const T* r = in + t * p.pst;
    const float dt = to_f(r[0]), x = to_f(r[p.ds]), bb = to_f(r[2 * p.ds]);
    const float d = softplus_acc(dt), sg = 1.f / (1.f + expf(-dt));
    const float g = to_f(dy[t * p.dst]) + c;
    const bool cut = rs && rs[t];
    c = cut ? 0.f : expf(d * A) * g;
    const float s = cut ? 0.f : c * hb[(int64_t)t * p.ds];
    dA = fmaf(s, d * A, dA);
    T* o = out + t * p.gst;
    o[0] = from_f<T>(fmaf(g * bb, x, s * A) * sg);
    o[p.ds] = from_f<T>(g * d * bb);
    o[2 * p.ds] = from_f<T>(g * d * x);
  }
  if (p.dh0) p.dh0[i] = c;
  p.dA_part[i] = dA;
}

// dA_log[j] = sum over the parts, in their order
__global__ void gated_scan_dA_kernel(const float* part, int parts, int ds, void* dA, int bf16) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= ds) return;
  float s = 0.f;
  for (int k = 0; k < parts; ++k) s += part[(int64_t)k * ds + j];
  if (bf16) static_cast<__nv_bfloat16*>(dA)[j] = __float2bfloat16_rn(s);
  else static_cast<float*>(dA)[j] = s;
}

template <typename T>
__global__ void __launch_bounds__(128) gated_step_kernel(const T* projs, int64_t psb, const void* A_log, int a_bf16,
                                                         const float* h, const uint8_t* reset, float* h_out, T* y,
                                                         int64_t ysb, int ds) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y;
  if (j >= ds) return;
  const T* r = projs + b * psb + j;
  const float A = -expf(ld_param(A_log, a_bf16, j));
  const float d = softplus_acc(to_f(r[0]));
  const float u = d * to_f(r[2 * ds]) * to_f(r[ds]);
  const int64_t i = (int64_t)b * ds + j;
  const float v = (reset && reset[b]) ? u : fmaf(expf(d * A), h[i], u);
  h_out[i] = v;
  y[b * ysb + j] = from_f<T>(v);
}

// largest grid and index ranges the kernels count in 32 bits
static int scan_check(const char* what, int dtype, int a_dtype, int64_t B, int64_t L, int64_t ds) {
  if ((dtype != HDC_F32 && dtype != HDC_BF16) || (a_dtype != HDC_F32 && a_dtype != HDC_BF16))
    return fail(HDC_E_DTYPE, "%s: dtype %d, A_log dtype %d", what, dtype, a_dtype);
  if (B < 0 || L < 0 || ds < 1 || B > 65535 || L > (int64_t(1) << 30) || ds > (int64_t(1) << 20))
    return fail(HDC_E_SHAPE, "%s: B=%lld in [0, 65535], L=%lld in [0, 2^30], d_state=%lld in [1, 2^20]", what,
                (long long)B, (long long)L, (long long)ds);
  return 0;
}

static bool off_type(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == HDC_F32 ? 3u : 1u)) != 0;
}

}  // namespace hdc

using namespace hdc;

extern "C" int64_t hdc_gated_scan_state_rows(void) { return kStateRows; }

extern "C" int hdc_gated_scan_fwd(int dtype, int a_dtype, const void* projs, int64_t proj_sb, int64_t proj_st,
                                  const void* A_log, const float* h0, const uint8_t* reset, void* y, int64_t y_sb,
                                  int64_t y_st, float* h_last, float* states, void* workspace, size_t workspace_bytes,
                                  int64_t B, int64_t L, int64_t ds, hdc_stream_t stream) {
  if (int e = scan_check("gated_scan", dtype, a_dtype, B, L, ds)) return e;
  if (B == 0) return HDC_OK;
  if (!A_log || (L > 0 && (!projs || !y))) return fail(HDC_E_NULL, "gated_scan: null pointer");
  if (off_type(projs, dtype) || off_type(y, dtype) || off_type(A_log, a_dtype) || off_type(h0, HDC_F32) ||
      off_type(h_last, HDC_F32) || off_type(states, HDC_F32))
    return fail(HDC_E_ALIGN, "gated_scan: a pointer is not aligned to its type");
  if (y_st < ds && L > 1) return fail(HDC_E_SHAPE, "gated_scan: y rows overlap (y_st=%lld)", (long long)y_st);
  if (workspace_bytes < hdc_gated_scan_workspace_bytes(B, L, ds))
    return fail(HDC_E_WORKSPACE, "gated_scan: workspace of %zu bytes is too small", workspace_bytes);
  ScanParams p{};
  p.projs = projs; p.psb = proj_sb; p.pst = proj_st; p.A_log = A_log; p.a_bf16 = a_dtype == HDC_BF16;
  p.h0 = h0; p.reset = reset; p.y = y; p.ysb = y_sb; p.yst = y_st; p.h_last = h_last; p.states = states;
  p.B = (int)B; p.L = (int)L; p.ds = (int)ds; p.NT = (int)((L + kStateRows - 1) / kStateRows);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)((B * ds + 127) / 128);
  if (dtype == HDC_F32) gated_scan_fwd_kernel<float><<<grid, 128, 0, s>>>(p);
  else gated_scan_fwd_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  return launch_status("gated_scan_fwd_kernel");
}

extern "C" size_t hdc_gated_scan_workspace_bytes(int64_t B, int64_t L, int64_t ds) { return 0; }

extern "C" size_t hdc_gated_scan_bwd_workspace_bytes(int64_t B, int64_t L, int64_t ds) {
  if (B < 1 || L < 0 || ds < 1) return 0;
  return (size_t)B * ds * 4 * (1 + L);
}

extern "C" int hdc_gated_scan_bwd(int dtype, int a_dtype, const void* projs, int64_t proj_sb, int64_t proj_st,
                                  const void* A_log, const float* states, const uint8_t* reset, const void* dy,
                                  int64_t dy_sb, int64_t dy_st, const float* dh_last, void* dprojs, int64_t dp_sb,
                                  int64_t dp_st, void* dA_log, float* dh0, void* workspace, size_t workspace_bytes,
                                  int64_t B, int64_t L, int64_t ds, hdc_stream_t stream) {
  if (int e = scan_check("gated_scan_bwd", dtype, a_dtype, B, L, ds)) return e;
  if (!A_log || !dA_log || (B > 0 && L > 0 && (!projs || !states || !dy || !dprojs)))
    return fail(HDC_E_NULL, "gated_scan_bwd: null pointer");
  if (off_type(projs, dtype) || off_type(dy, dtype) || off_type(dprojs, dtype) || off_type(A_log, a_dtype) ||
      off_type(dA_log, a_dtype) || off_type(states, HDC_F32) || off_type(dh_last, HDC_F32) || off_type(dh0, HDC_F32) ||
      off_type(workspace, HDC_F32))
    return fail(HDC_E_ALIGN, "gated_scan_bwd: a pointer is not aligned to its type");
  if (dp_st < 3 * ds && L > 1)
    return fail(HDC_E_SHAPE, "gated_scan_bwd: dprojs rows overlap (dp_st=%lld)", (long long)dp_st);
  const size_t need = hdc_gated_scan_bwd_workspace_bytes(B, L, ds);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(HDC_E_WORKSPACE, "gated_scan_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  ScanParams p{};
  p.projs = projs; p.psb = proj_sb; p.pst = proj_st; p.A_log = A_log; p.a_bf16 = a_dtype == HDC_BF16;
  p.reset = reset; p.states = const_cast<float*>(states); p.dy = dy; p.dsb = dy_sb; p.dst = dy_st;
  p.dh_last = dh_last; p.dprojs = dprojs; p.gsb = dp_sb; p.gst = dp_st; p.dh0 = dh0;
  p.dA_part = static_cast<float*>(workspace); p.hbuf = p.dA_part + B * ds;
  p.B = (int)B; p.L = (int)L; p.ds = (int)ds; p.NT = (int)((L + kStateRows - 1) / kStateRows);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  if (B > 0) {
    const unsigned grid = (unsigned)((B * ds + 127) / 128);
    if (dtype == HDC_F32) gated_scan_bwd_kernel<float><<<grid, 128, 0, s>>>(p);
    else gated_scan_bwd_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
    if (int e = launch_status("gated_scan_bwd_kernel")) return e;
  }
  gated_scan_dA_kernel<<<(unsigned)((ds + 127) / 128), 128, 0, s>>>(p.dA_part, (int)B, (int)ds, dA_log, p.a_bf16);
  return launch_status("gated_scan_dA_kernel");
}

extern "C" int hdc_gated_step(int dtype, int a_dtype, const void* projs, int64_t proj_sb, const void* A_log,
                              const float* h, const uint8_t* reset, float* h_out, void* y, int64_t y_sb, int64_t B,
                              int64_t ds, hdc_stream_t stream) {
  if (int e = scan_check("gated_step", dtype, a_dtype, B, 1, ds)) return e;
  if (B == 0) return HDC_OK;
  if (!projs || !A_log || !h || !h_out || !y) return fail(HDC_E_NULL, "gated_step: null pointer");
  if (off_type(projs, dtype) || off_type(y, dtype) || off_type(A_log, a_dtype) || off_type(h, HDC_F32) ||
      off_type(h_out, HDC_F32))
    return fail(HDC_E_ALIGN, "gated_step: a pointer is not aligned to its type");
  if (y_sb < ds && B > 1) return fail(HDC_E_SHAPE, "gated_step: y rows overlap (y_sb=%lld)", (long long)y_sb);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((ds + 127) / 128), (unsigned)B);
  const int ab = a_dtype == HDC_BF16;
  if (dtype == HDC_F32)
    gated_step_kernel<float><<<grid, 128, 0, s>>>(static_cast<const float*>(projs), proj_sb, A_log, ab, h, reset,
                                                  h_out, static_cast<float*>(y), y_sb, (int)ds);
  else
    gated_step_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(static_cast<const __nv_bfloat16*>(projs), proj_sb, A_log, ab,
                                                          h, reset, h_out, static_cast<__nv_bfloat16*>(y), y_sb,
                                                          (int)ds);
  return launch_status("gated_step_kernel");
}
