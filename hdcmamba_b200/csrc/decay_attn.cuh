// Linear attention with a decay for each head: what its kernels share.
//
// Forward, per batch and head with decay e = exp(g):  S_t = e S_{t-1} + k_t v_t',  o_t = scale q_t' S_t.
// Its gradient, with G_t the gradient of S_t (dS behind the last token):
//   dq_t = scale S_t do_t,   G_t = e G_{t+1} + scale q_t do_t',   dk_t = G_t v_t,   dv_t = G_t' k_t,   dS_0 = e G_1.
// All four outputs have one form, which is what a pass computes:
//   out_t = x_t' M_t,   M a decayed sum of y_t z_t' forwards or backwards in time:
//   o (x, y, z) = (q, k, v);  dq = (do, v, k), M = S';  dv backwards = (k, q, do), M = G;  dk backwards = (v, do, q), M = G'.
//
// Time is cut into chunks of 64 tokens (128 in decay_attn_tc.cu) and segments of whole chunks.  With R the state that enters a chunk
// of n tokens (i, j local indices),
//   out_i = si in(i) x_i' R + sum_j sa e^|i-j| (x_i' y_j) z_j   over j <= i (backwards j >= i),
//   R <- e^n R + sum_j su up(j) y_j z_j',
// with in(i) = e^(i+1), up(j) = e^(n-1-j) forwards and in(i) = e^(n-1-i), up(j) = e^(j+1) backwards.
// A first kernel sums every segment's own state, a second joins the segments, a third writes the
// outputs; a sequence of one segment needs the third alone, which then writes the state behind it too.  No
// kernel waits for another CTA, and results do not depend on timing.  (Joining up to eight segments in the third
// kernel instead costs it registers and time: 8 x 4096 x 16 heads of 64 with gradient 544 us for 457.)
#pragma once
#include "common.cuh"

namespace hdc {

constexpr int kAttnChunk = 64;

struct AttnView {
  const void* p;
  int64_t sb, st, sh;  // strides of batch, token and head, in elements; the head's elements lie side by side
};

struct AttnPass {
  AttnView x, y, z, out;
  float* states;  // [B * H][nseg][D * D]: the state that enters each segment (the sums' kernel: each segment's own)
  // a sequence of one segment (p.nseg == 1): the state that enters it (NULL: zeros) and, unless NULL, where the one
  // that leaves it goes
  const float* from;
  float* to;
  int transposed, backwards;
  float sa, si, su;
  int out_vec;  // out takes 16-byte stores
};

struct AttnParams {
  AttnPass pass[3];
  const float* g;
  int H, L, D, nseg, seg;  // seg: tokens of a segment, whole chunks
  int wide;                // segments of whole 128 tokens, outputs by the tcgen05 kernel where strides allow it
};

// exp(g d), 1 for d = 0 whatever g is
__device__ __forceinline__ float decay_pow(float g, int d) { return d == 0 ? 1.f : expf(g * (float)d); }

// the state that enters a CTA's segment, or NULL for zeros
__device__ __forceinline__ const float* entering(const AttnParams& p, const AttnPass& a, int64_t bh, int seg) {
  const int64_t DD = (int64_t)p.D * p.D;
  return p.nseg > 1 ? a.states + (bh * p.nseg + seg) * DD : a.from ? a.from + bh * DD : nullptr;
}

// Tokens that are not finite.  The products of a chunk's tokens with one another have zeros behind the causal mask, and
// zero times infinity is NaN: a token would reach outputs before it (behind it, backwards).  The outputs' kernels look at
// what they have computed, some ten instructions a chunk, and where an output of a segment is not finite its CTA
// computes those outputs again by the recurrence, token by token, which knows no mask: M is the state that enters the
// segment, in shared memory, and four lanes take a column.  Once every column of M holds a value that is not finite, no
// output behind it is finite by the definition either, and the rest stays as it is: a sequence that is NaN throughout costs
// its segments a token each.  (Guards around the products themselves, zeros in their place, cost 3 to 15% of the outputs'
// time.  The recurrence takes some 2.5 us a token of 64, for outputs whose products overflow in the check, too.)
__device__ __forceinline__ void state_for_recurrence(const AttnParams& p, const AttnPass& a, int64_t bh, int seg, float* M) {
  const float* state = entering(p, a, bh, seg);
  for (int i = threadIdx.x; i < p.D * p.D; i += blockDim.x) {
    const int r = i / p.D, c = i % p.D;  // of the state in memory
    M[a.transposed ? c * p.D + r : i] = state ? state[i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void by_recurrence(const AttnParams& p, const AttnPass& a, int64_t bh, int seg, float* M) {
  const int D = p.D, back = a.backwards, b = (int)(bh / p.H), h = (int)(bh % p.H), lane = threadIdx.x % 4;
  const int begin = seg * p.seg, end = min(p.L, begin + p.seg);
  const T* const x0 = static_cast<const T*>(a.x.p) + b * a.x.sb + h * a.x.sh;
  const T* const y0 = static_cast<const T*>(a.y.p) + b * a.y.sb + h * a.y.sh;
  const T* const z0 = static_cast<const T*>(a.z.p) + b * a.z.sb + h * a.z.sh;
  T* const out0 = static_cast<T*>(const_cast<void*>(a.out.p)) + b * a.out.sb + h * a.out.sh;
  const float e = decay_pow(p.g[h], 1);
#pragma unroll 1
  for (int i = begin; i < end; ++i) {
    const int64_t t = back ? begin + end - 1 - i : i;
    const T *x = x0 + t * a.x.st, *y = y0 + t * a.y.st;
    bool lost = true;  // the thread's columns
#pragma unroll 1
    for (int c0 = 0; c0 < D; c0 += blockDim.x / 4) {
      const int c = c0 + threadIdx.x / 4;
      float sum = 0.f, odd = 0.f;
      if (c < D) {
        const float z = a.su * to_f(z0[t * a.z.st + c]);
        // forwards a token decays what was there before it, backwards what goes on to the one before it
#pragma unroll 4
        for (int r = lane; r < D; r += 4) {
          float m = fmaf(to_f(y[r]), z, back ? M[r * D + c] : e * M[r * D + c]);
          sum = fmaf(to_f(x[r]), m, sum);
          m = back ? e * m : m;
          odd = fmaf(m, 0.f, odd);
          M[r * D + c] = m;
        }
      }
#pragma unroll
      for (int k = 1; k < 4; k *= 2) {
        sum += __shfl_xor_sync(~0u, sum, k);
        odd += __shfl_xor_sync(~0u, odd, k);
      }
      if (lane == 0 && c < D) {
        T* o = out0 + t * a.out.st + c;
        if (!(fabsf(to_f(*o)) <= 3.4028235e38f)) *o = from_f<T>(a.si * sum);  // finite ones are right as they are
      }
      lost = lost && (c >= D || odd != 0.f);
    }
    if ((i - begin) % 16 == 0 && __syncthreads_and(lost)) return;
  }
}
// of a pair of sums of products of two outputs
__device__ __forceinline__ bool all_finite(uint64_t sums) {
  float s0, s1;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(s0), "=f"(s1) : "l"(sums));
  return fabsf(s0 + s1) <= 3e38f;
}

// csrc/decay_attn_f32.cu, csrc/decay_attn_bf16.cu: the segments' own states (pass 0), and passes' outputs
int attn_sums_f32(AttnParams& p, int64_t bh, cudaStream_t s);
int attn_out_f32(AttnParams& p, int64_t bh, int passes, cudaStream_t s);
int attn_sums_bf16(AttnParams& p, int64_t bh, cudaStream_t s);
int attn_out_bf16(AttnParams& p, int64_t bh, int passes, cudaStream_t s);
// csrc/decay_attn_tc.cu: outputs of several segments of whole 128 tokens (but for the last one's end), heads of at
// most 64 whose rows allow 16-byte copies; false where a tensor's strides do not suit it
bool attn_out_tc(const AttnParams& p, int64_t bh, int passes, cudaStream_t s, int* status);

}  // namespace hdc
