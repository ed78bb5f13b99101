// Decayed linear attention: entry points, the joining of segments, and the single-token step.
// The mathematics stands in decay_attn.cuh.
#include <type_traits>

#include "decay_attn.cuh"
#include "vec.cuh"

namespace hdc {

// ---------------------------------------------------------------- segments joined
// states[n] holds segment n's own sum; afterwards the state that enters it: run_{n+1} = e^len run_n + own_n
// in the order of the pass, from `from` (or zeros); `to` (or NULL) takes the state behind the last one.
// A thread per V elements of a state walks the segments; the loads of kAhead of them are in flight.
template <int V>
__global__ void __launch_bounds__(128) attn_join_kernel(float* states, const float* from, float* to, const float* g,
                                                        int H, int L, int DD, int nseg, int seg, int backwards) {
  constexpr int kAhead = 8;
  const int64_t bh = blockIdx.x;
  const int i = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (i >= DD) return;
  let_next_start();
  const float d = g[bh % H];
  const float whole = decay_pow(d, seg), rest = decay_pow(d, L - (nseg - 1) * seg);
  float run[V];
#pragma unroll
  for (int e = 0; e < V; ++e) run[e] = from ? from[bh * DD + i + e] : 0.f;
  wait_for_previous();
  float* s = states + bh * nseg * DD + i;
  for (int n0 = 0; n0 < nseg; n0 += kAhead) {
    float own[kAhead][V];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (n0 + k < nseg) {
        const float* src = s + (int64_t)(backwards ? nseg - 1 - n0 - k : n0 + k) * DD;
        if constexpr (V == 4) *reinterpret_cast<float4*>(own[k]) = *reinterpret_cast<const float4*>(src);
        else own[k][0] = src[0];
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int n = backwards ? nseg - 1 - n0 - k : n0 + k;
      if (n0 + k < nseg) {
        float* dst = s + (int64_t)n * DD;
        if constexpr (V == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(run);
        else dst[0] = run[0];
        const float keep = n == nseg - 1 ? rest : whole;
#pragma unroll
        for (int e = 0; e < V; ++e) run[e] = fmaf(keep, run[e], own[k][e]);
      }
    }
  }
  if (!to) return;
#pragma unroll
  for (int e = 0; e < V; ++e) to[bh * DD + i + e] = run[e];
}

// ---------------------------------------------------------------- one token
// S <- e S + k v', o = scale q' S.  256 threads take whole states, one after another in memory: CG lanes of 4
// columns side by side, the others every RG-th row, their loads in flight at once; the rows' parts of o are added in
// shared memory.  Bound by the state's traffic (read and written once) at large batches, by one load's latency
// and the launch at small ones: 12 states of 64 x 64 2.6 us.
template <typename T, int CG, bool VEC>
__global__ void __launch_bounds__(256) attn_step_kernel(AttnView q, AttnView k, AttnView v, AttnView o, const float* g,
                                                        const float* state, float* state_out, float scale, int H,
                                                        int D, int64_t states) {
  constexpr int RG = CG == 32 ? 8 : 16, PER = 256 / (CG * RG), ROWS = CG * 4 / RG, AHEAD = ROWS < 8 ? ROWS : 8;
  __shared__ float part[PER][RG][CG * 4 + 4];
  const int own = threadIdx.x / (CG * RG), rg = threadIdx.x / CG % RG, c = threadIdx.x % CG * 4;
  const int64_t bh = (int64_t)blockIdx.x * PER + own;
  const bool there = bh < states;
  const int b = there ? (int)(bh / H) : 0, h = there ? (int)(bh % H) : 0;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (there && c < D) {
    const T* qp = static_cast<const T*>(q.p) + b * q.sb + h * q.sh;
    const T* kp = static_cast<const T*>(k.p) + b * k.sb + h * k.sh;
    const T* vp = static_cast<const T*>(v.p) + b * v.sb + h * v.sh;
    const float* s = state + bh * D * D + c;
    float* t = state_out + bh * D * D + c;
    const int cols = min(4, D - c);
    const float e = expf(g[h]);
    float vv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] = j < cols ? to_f(vp[c + j]) : 0.f;
#pragma unroll
    for (int i0 = 0; i0 < ROWS; i0 += AHEAD) {
      float x[AHEAD][4], kk[AHEAD], qq[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int r = rg + (i0 + i) * RG;
        if (r >= D) continue;
        if constexpr (VEC) {
          *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(s + r * D);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[i][j] = j < cols ? s[r * D + j] : 0.f;
        }
        kk[i] = to_f(kp[r]);
        qq[i] = to_f(qp[r]);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int r = rg + (i0 + i) * RG;
        if (r >= D) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[i][j] = fmaf(e, x[i][j], kk[i] * vv[j]);
          acc[j] = fmaf(qq[i], x[i][j], acc[j]);
        }
        if constexpr (VEC) {
          *reinterpret_cast<float4*>(t + r * D) = *reinterpret_cast<const float4*>(x[i]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < cols) t[r * D + j] = x[i][j];
        }
      }
    }
  }
  *reinterpret_cast<float4*>(&part[own][rg][c]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  const int col = threadIdx.x % (CG * RG);
  if (!there || col >= D) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < RG; ++i) sum += part[own][i][col];
  static_cast<T*>(const_cast<void*>(o.p))[b * o.sb + h * o.sh + col] = from_f<T>(scale * sum);
}

// ---------------------------------------------------------------- plans and checks
// Whether the outputs come from the tcgen05 kernel: heads of 33 to 64 in bf16, and enough tokens that its longer
// chunks pay.  Forward in us with it and without: 12 heads 1024 tokens 18 and 17, 2048 21 and 21, 16384 56 and 56; 4 heads
// 1024 tokens 15 and 12, 4096 17 and 20; 32 heads 768 tokens 21 and 19, 1024 21 and 23, 16384 119 and 134; 128 heads 4096
// tokens 135 and 147.
static bool attn_wide(int dtype, int64_t heads, int64_t chunks, int64_t D) {
  return dtype == HDC_BF16 && D > 32 && D <= 64 && (chunks >= 32 || heads * chunks >= 512);
}

// Tokens of a segment, a function of the sizes alone (so that a forward and its gradient agree, and results do not
// depend on the device's SM count): enough segments for the CTAs that 148 SMs hold, or one where a single launch
// over all chunks takes no longer than the three over segments.  Forward in us, one segment and several (bf16:
// 16 heads of 32 128 tokens 7 and 13, 257 12 and 12, 512 17 and 13; 128 heads of 64 257 tokens 19 and 29, 1024 45 and 53;
// 4 heads of 128 128 tokens 19 and 25, 257 35 and 25.  fp32: 12 heads of 64 64 tokens 19 and 19, 128 33 and 25; 128
// heads of 64 257 tokens 72 and 78, 384 90 and 78).
static int64_t attn_seg(int dtype, int64_t B, int64_t L, int64_t H, int64_t D) {
  const int64_t chunks = (L + kAttnChunk - 1) / kAttnChunk, heads = B * H;
  if (chunks < 1 || heads < 1) return kAttnChunk;
  const bool wide = attn_wide(dtype, heads, chunks, D);
  const int64_t ctas = 148 * (wide ? 2 : 3);
  const int64_t alone = dtype == HDC_F32 ? 1 + heads / 32 : D <= 64 ? 4 + heads / 10 : 2 + heads / 20;
  int64_t want = chunks <= alone ? 1 : ctas / heads;
  if (want < 1) want = 1;
  if (want > chunks) want = chunks;
  if (wide && want > 1) {  // whole 128 tokens
    const int64_t pairs = (chunks + 1) / 2;
    if (want > pairs) want = pairs;
    return (pairs + want - 1) / want * 2 * kAttnChunk;
  }
  return (chunks + want - 1) / want * kAttnChunk;
}
static int64_t attn_nseg(int dtype, int64_t B, int64_t L, int64_t H, int64_t D) {
  const int64_t seg = attn_seg(dtype, B, L, H, D);
  return (L + seg - 1) / seg;
}

static int attn_check(const char* what, int dtype, int64_t B, int64_t L, int64_t H, int64_t D) {
  if (dtype != HDC_F32 && dtype != HDC_BF16) return fail(HDC_E_DTYPE, "%s: dtype %d", what, dtype);
  if (B < 0 || L < 0 || H < 1 || D < 1 || D > 128 || L > (int64_t(1) << 30) || B > (int64_t(1) << 30) ||
      H > (int64_t(1) << 20) || B * H * attn_nseg(dtype, B, L, H, D) >= (int64_t(1) << 31))
    return fail(HDC_E_SHAPE, "%s: B=%lld, L=%lld in [0, 2^30], H=%lld in [1, 2^20], D=%lld in [1, 128]", what,
                (long long)B, (long long)L, (long long)H, (long long)D);
  return 0;
}

static bool off_type(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == HDC_F32 ? 3u : 1u)) != 0;
}

// a tensor's view; the stride of a dimension of one does not count
static AttnView view_of(const void* p, int64_t sb, int64_t st, int64_t sh, int64_t B, int64_t L, int64_t H) {
  return {p, B > 1 ? sb : 0, L > 1 ? st : 0, H > 1 ? sh : 0};
}

// the heads' rows [B, L, H] of D elements of an output lie apart: by growing stride, each steps over all
// that the ones before reach
static bool heads_apart(const AttnView& v, int64_t B, int64_t L, int64_t H, int64_t D) {
  int64_t n[3] = {B, L, H}, s[3] = {v.sb, v.st, v.sh};
  for (int i = 0; i < 3; ++i)
    if (n[i] < 2) s[i] = 0;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (s[j] > s[j + 1]) {
        int64_t t = s[j]; s[j] = s[j + 1]; s[j + 1] = t;
        t = n[j]; n[j] = n[j + 1]; n[j + 1] = t;
      }
  int64_t reach = D;
  for (int i = 0; i < 3; ++i) {
    if (n[i] < 2) continue;
    if (s[i] < reach) return false;
    reach += (n[i] - 1) * s[i];
  }
  return true;
}

static int join(float* states, const float* from, float* to, const AttnParams& p, int64_t bh, int backwards,
                cudaStream_t s) {
  const int DD = p.D * p.D;
  const bool vec = p.D % 2 == 0 && aligned16(states) && aligned16(from);
  const int per = vec ? 512 : 128;
  const dim3 grid((unsigned)bh, (unsigned)((DD + per - 1) / per));
  launch_dependent(vec ? attn_join_kernel<4> : attn_join_kernel<1>, grid, 128, 0, s, states, from, to, p.g, p.H, p.L, DD, p.nseg,
                   p.seg, backwards);
  return launch_status("attn_join_kernel");
}

static int copy_state(const char* what, const float* from, float* to, int64_t n, cudaStream_t s) {
  if (!to) return HDC_OK;
  const cudaError_t e = from ? cudaMemcpyAsync(to, from, (size_t)n * 4, cudaMemcpyDeviceToDevice, s)
                             : cudaMemsetAsync(to, 0, (size_t)n * 4, s);
  return e == cudaSuccess ? HDC_OK : fail((int)e, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace hdc

using namespace hdc;

extern "C" int64_t hdc_decay_attn_state_slots(int dtype, int64_t B, int64_t L, int64_t H, int64_t D) {
  return L < 1 || B < 1 || H < 1 || D < 1 ? 0 : attn_nseg(dtype, B, L, H, D);
}

static void plan(AttnParams& p, int dtype, const float* log_decay, int64_t B, int64_t L, int64_t H, int64_t D) {
  p.g = log_decay; p.H = (int)H; p.L = (int)L; p.D = (int)D;
  p.seg = (int)attn_seg(dtype, B, L, H, D); p.nseg = (int)attn_nseg(dtype, B, L, H, D);
  p.wide = p.nseg > 1 && attn_wide(dtype, B * H, (L + kAttnChunk - 1) / kAttnChunk, D);
}

extern "C" int hdc_decay_attn_fwd(int dtype, const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k,
                                  int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st,
                                  int64_t v_sh, const float* log_decay, const float* state_in, float scale, void* o,
                                  int64_t o_sb, int64_t o_st, int64_t o_sh, float* state_out, float* states, int64_t B,
                                  int64_t L, int64_t H, int64_t D, hdc_stream_t stream) {
  if (int e = attn_check("decay_attn", dtype, B, L, H, D)) return e;
  if (B == 0) return HDC_OK;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  if (off_type(q, dtype) || off_type(k, dtype) || off_type(v, dtype) || off_type(o, dtype) ||
      off_type(log_decay, HDC_F32) || off_type(state_in, HDC_F32) || off_type(state_out, HDC_F32) ||
      off_type(states, HDC_F32))
    return fail(HDC_E_ALIGN, "decay_attn: a pointer is not aligned to its type");
  if (L == 0) return copy_state("decay_attn", state_in, state_out, B * H * D * D, s);
  AttnParams p{};
  plan(p, dtype, log_decay, B, L, H, D);
  if (!q || !k || !v || !o || !log_decay || (!states && p.nseg > 1)) return fail(HDC_E_NULL, "decay_attn: null pointer");
  auto view = [&](const void* t, int64_t sb, int64_t st, int64_t sh) { return view_of(t, sb, st, sh, B, L, H); };
  const AttnView Q = view(q, q_sb, q_st, q_sh), K = view(k, k_sb, k_st, k_sh), V = view(v, v_sb, v_st, v_sh),
                 O = view(o, o_sb, o_st, o_sh);
  if (!heads_apart(O, B, L, H, D)) return fail(HDC_E_SHAPE, "decay_attn: rows of o overlap");
  p.pass[0] = {Q, K, V, O, states, state_in, state_out, 0, 0, scale, scale, 1.f};
  const int64_t bh = B * H;
  const bool f32 = dtype == HDC_F32;
  if (p.nseg > 1) {
    if (int e = f32 ? attn_sums_f32(p, bh, s) : attn_sums_bf16(p, bh, s)) return e;
    if (int e = join(states, state_in, state_out, p, bh, 0, s)) return e;
  } else if (states) {  // what enters the one segment, for the gradient
    if (int e = copy_state("decay_attn", state_in, states, bh * D * D, s)) return e;
  }
  return f32 ? attn_out_f32(p, bh, 1, s) : attn_out_bf16(p, bh, 1, s);
}

extern "C" size_t hdc_decay_attn_bwd_workspace_bytes(int dtype, int64_t B, int64_t L, int64_t H, int64_t D) {
  const int64_t slots = hdc_decay_attn_state_slots(dtype, B, L, H, D);
  return slots > 1 ? (size_t)(B * H * slots) * D * D * 4 : 0;
}

extern "C" int hdc_decay_attn_bwd(int dtype, const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k,
                                  int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st,
                                  int64_t v_sh, const void* dout, int64_t do_sb, int64_t do_st, int64_t do_sh,
                                  const float* log_decay, const float* states, const float* dstate_out, float scale,
                                  void* dq, int64_t dq_sb, int64_t dq_st, int64_t dq_sh, void* dk, int64_t dk_sb,
                                  int64_t dk_st, int64_t dk_sh, void* dv, int64_t dv_sb, int64_t dv_st, int64_t dv_sh,
                                  float* dstate_in, void* workspace, size_t workspace_bytes, int64_t B, int64_t L,
                                  int64_t H, int64_t D, hdc_stream_t stream) {
  if (int e = attn_check("decay_attn_bwd", dtype, B, L, H, D)) return e;
  if (B == 0) return HDC_OK;
  auto s = reinterpret_cast<cudaStream_t>(stream);
  if (off_type(q, dtype) || off_type(k, dtype) || off_type(v, dtype) || off_type(dout, dtype) || off_type(dq, dtype) ||
      off_type(dk, dtype) || off_type(dv, dtype) || off_type(log_decay, HDC_F32) || off_type(states, HDC_F32) ||
      off_type(dstate_out, HDC_F32) || off_type(dstate_in, HDC_F32))
    return fail(HDC_E_ALIGN, "decay_attn_bwd: a pointer is not aligned to its type");
  if (L == 0) return copy_state("decay_attn_bwd", dstate_out, dstate_in, B * H * D * D, s);
  if (!q || !k || !v || !dout || !dq || !dk || !dv || !log_decay || !states)
    return fail(HDC_E_NULL, "decay_attn_bwd: null pointer");
  const size_t need = hdc_decay_attn_bwd_workspace_bytes(dtype, B, L, H, D);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(HDC_E_WORKSPACE, "decay_attn_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!aligned16(workspace)) return fail(HDC_E_ALIGN, "decay_attn_bwd: the workspace is not 16-byte aligned");
  auto view = [&](const void* t, int64_t sb, int64_t st, int64_t sh) { return view_of(t, sb, st, sh, B, L, H); };
  const AttnView Q = view(q, q_sb, q_st, q_sh), K = view(k, k_sb, k_st, k_sh), V = view(v, v_sb, v_st, v_sh),
                 DO = view(dout, do_sb, do_st, do_sh);
  const AttnView DQ = view(dq, dq_sb, dq_st, dq_sh), DK = view(dk, dk_sb, dk_st, dk_sh), DV = view(dv, dv_sb, dv_st, dv_sh);
  if (!heads_apart(DQ, B, L, H, D) || !heads_apart(DK, B, L, H, D) || !heads_apart(DV, B, L, H, D))
    return fail(HDC_E_SHAPE, "decay_attn_bwd: rows of dq, dk or dv overlap");
  float* grads = static_cast<float*>(workspace);
  AttnParams p{};
  plan(p, dtype, log_decay, B, L, H, D);
  const int64_t bh = B * H;
  const bool f32 = dtype == HDC_F32;
  p.pass[0] = {K, Q, DO, DV, grads, dstate_out, dstate_in, 0, 1, scale, 1.f, scale};
  p.pass[1] = {V, DO, Q, DK, grads, dstate_out, nullptr, 1, 1, scale, 1.f, scale};
  p.pass[2] = {DO, V, K, DQ, const_cast<float*>(states), states, nullptr, 1, 0, scale, scale, 1.f};
  if (p.nseg > 1) {
    if (int e = f32 ? attn_sums_f32(p, bh, s) : attn_sums_bf16(p, bh, s)) return e;
    if (int e = join(grads, dstate_out, dstate_in, p, bh, 1, s)) return e;
  }
  return f32 ? attn_out_f32(p, bh, 3, s) : attn_out_bf16(p, bh, 3, s);
}

extern "C" int hdc_decay_attn_step(int dtype, const void* q, int64_t q_sb, int64_t q_sh, const void* k, int64_t k_sb,
                                   int64_t k_sh, const void* v, int64_t v_sb, int64_t v_sh, const float* log_decay,
                                   const float* state, float scale, void* o, int64_t o_sb, int64_t o_sh,
                                   float* state_out, int64_t B, int64_t H, int64_t D, hdc_stream_t stream) {
  if (int e = attn_check("decay_attn_step", dtype, B, 1, H, D)) return e;
  if (B == 0) return HDC_OK;
  if (!q || !k || !v || !o || !log_decay || !state || !state_out)
    return fail(HDC_E_NULL, "decay_attn_step: null pointer");
  if (off_type(q, dtype) || off_type(k, dtype) || off_type(v, dtype) || off_type(o, dtype) ||
      off_type(log_decay, HDC_F32) || off_type(state, HDC_F32) || off_type(state_out, HDC_F32))
    return fail(HDC_E_ALIGN, "decay_attn_step: a pointer is not aligned to its type");
  const AttnView Q{q, q_sb, 0, q_sh}, K{k, k_sb, 0, k_sh}, V{v, v_sb, 0, v_sh}, O{o, o_sb, 0, o_sh};
  if (!heads_apart(O, B, 1, H, D)) return fail(HDC_E_SHAPE, "decay_attn_step: rows of o overlap");
  auto s = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = D % 4 == 0 && aligned16(state) && aligned16(state_out);
  const int64_t n = B * H;
  auto launch = [&](auto kernel, int per) {
    kernel<<<(unsigned)((n + per - 1) / per), 256, 0, s>>>(Q, K, V, O, log_decay, state, state_out, scale, (int)H, (int)D, n);
  };
  auto sized = [&](auto t, auto vec_) {
    using T = decltype(t);
    constexpr bool kVec = decltype(vec_)::value;
    if (D <= 16) launch(attn_step_kernel<T, 4, kVec>, 4);
    else if (D <= 32) launch(attn_step_kernel<T, 8, kVec>, 2);
    else if (D <= 64) launch(attn_step_kernel<T, 16, kVec>, 1);
    else launch(attn_step_kernel<T, 32, kVec>, 1);
  };
  if (dtype == HDC_F32) vec ? sized(float(), std::true_type()) : sized(float(), std::false_type());
  else vec ? sized(__nv_bfloat16(), std::true_type()) : sized(__nv_bfloat16(), std::false_type());
  return launch_status("attn_step_kernel");
}
