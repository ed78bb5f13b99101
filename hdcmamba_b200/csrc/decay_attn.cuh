// Linear attention with a decay for each head: what its kernels share.
//
// Forward, per batch and head with decay e = exp(g):  S_t = e S_{t-1} + k_t v_t',  o_t = scale q_t' S_t.
// Its gradient, with G_t the gradient of S_t (dS behind the last token):
//   dq_t = scale S_t do_t,   G_t = e G_{t+1} + scale q_t do_t',   dk_t = G_t v_t,   dv_t = G_t' k_t,   dS_0 = e G_1.
// All four outputs have one form, which is what a pass computes:
//   out_t = x_t' M_t,   M a decayed sum of y_t z_t' forwards or backwards in time:
//   o (x, y, z) = (q, k, v);  dq = (do, v, k), M = S';  dv backwards = (k, q, do), M = G;  dk backwards = (v, do, q), M = G'.
//
// Time is cut into chunks of 64 tokens and those into segments.  With R the state that enters a chunk
// of n tokens (i, j local indices),
//   out_i = si in(i) x_i' R + sum_j sa e^|i-j| (x_i' y_j) z_j   over j <= i (backwards j >= i),
//   R <- e^n R + sum_j su up(j) y_j z_j',
// with in(i) = e^(i+1), up(j) = e^(n-1-j) forwards and in(i) = e^(n-1-i), up(j) = e^(j+1) backwards.
// A first kernel sums every segment's own state, a second joins the segments, a third writes the
// outputs; no kernel waits for another CTA, and results do not depend on timing.
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
  int transposed, backwards;
  float sa, si, su;
  int out_vec;  // out takes 16-byte stores
};

struct AttnParams {
  AttnPass pass[3];
  const float* g;
  int H, L, D, nseg, seg;  // seg: tokens of a segment, whole chunks
};

// exp(g d), 1 for d = 0 whatever g is
__device__ __forceinline__ float decay_pow(float g, int d) { return d == 0 ? 1.f : expf(g * (float)d); }

// csrc/decay_attn_f32.cu, csrc/decay_attn_bf16.cu: the segments' own states (pass 0), and passes' outputs
int attn_sums_f32(AttnParams& p, int64_t bh, cudaStream_t s);
int attn_out_f32(AttnParams& p, int64_t bh, int passes, cudaStream_t s);
int attn_sums_bf16(AttnParams& p, int64_t bh, cudaStream_t s);
int attn_out_bf16(AttnParams& p, int64_t bh, int passes, cudaStream_t s);

}  // namespace hdc
