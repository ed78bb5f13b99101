// Decayed linear attention of bf16 tensors on the tensor cores (mma.sync m16n8k16, fp32 sums).
//
// A CTA walks the 64-token chunks of one segment of one batch and head.  The state R stays in fp32 in the
// accumulators of the warps, 16 rows each; a copy rounded to bf16 goes through shared memory to the product
// x R of the next chunk.  Per chunk and warp (16 tokens of outputs):
//   O = in(i) X R;  S = X Y' (the tiles on and below the diagonal);  P = decay * S;  O += P Z;  R = e^n R + (up Y)' Z.
// S becomes P in registers: an accumulator tile has the layout of the next product's operand.
//
// Roundings.  P and the copy of R are rounded to bf16 once, as the result is; sums and states stay fp32.  The
// weighted tokens up(j) y_j would add a third rounding to every state: they are split into two bf16 parts (2^-17), and
// into three (2^-25) where the fp32 state that the caller gets is made of them: in a sequence of one segment, and in
// those segments' sums of which more than 2^-8 is left at the end of the pass (the others' 2^-17 is 2^-25 there; a
// quarter was too much, where the few tokens behind it happened to be small).  Sums for such a state are also added up
// chunk by chunk outside the tensor cores, whose own sums of many steps lose low bits one-sidedly.
//
// Bound by mma.sync: one m16n8k16 takes 16 cycles of a sub-partition (512 multiply-adds per clock and SM), so the
// 136 of a chunk and warp come to 52 us for 32768 x 12 heads of 64, and the 64 to 96 of the sums to 23 to 34; measured
// 63 and 33, at 201 and 101 MB (31 and 15 us).  (Outputs of many tokens with heads of 33 to 64: decay_attn_tc.cu.)  Three chunks in flight instead of two change nothing; all four
// products with a whole square instead of its causal part cost 6 us more.
#include <atomic>

#include "decay_attn.cuh"
#include "vec.cuh"

namespace hdc {

using bf16 = __nv_bfloat16;

// A tile in shared memory: rows of DP values and 16 bytes more, so that eight neighbouring rows of one 16-byte
// unit lie in different banks and every address is a lane's base and a constant.
template <int DP> constexpr int kPitch = DP * 2 + 16;

__device__ __forceinline__ uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // from zero
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// pairs of fp32 values: one instruction for two
__device__ __forceinline__ void scale2(float& x, float& y, float f, float h) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(x, y)), "l"(pair_bits(f, h)));
  bits_pair(r, x, y);
}
__device__ __forceinline__ void fma2(uint64_t& s, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(s) : "l"(a), "l"(b));
}
// (x, y) minus the two bf16 values of v
__device__ __forceinline__ void less2(float& x, float& y, uint32_t v) {
  uint64_t r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(x, y)), "l"(pair_bits(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u))));
  bits_pair(r, x, y);
}
template <bool FIRST, typename A, typename B> __device__ __forceinline__ auto& first_if(A& a, B& b) {
  if constexpr (FIRST) return a;
  else return b;
}

// What a kernel computes: segments' sums; outputs; outputs and the state behind a sequence of one segment.
constexpr int kSums = 0, kOutputs = 1, kWhole = 2;

template <int DP> struct AttnShape {
  static constexpr int kWarps = DP == 128 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTile = kAttnChunk * kPitch<DP>;           // bytes of a tile
  static constexpr int kStateCols = DP == 32 ? 16 : DP;           // a warp's columns of the state (16 rows)
  static constexpr int kOutCols = DP == 128 ? 64 : DP;            // a warp's columns of the outputs (16 tokens)
  static constexpr int tiles(bool out) { return out ? 3 : 2; }    // of a stage
  static constexpr int smem(bool out) { return 2 * tiles(out) * kTile + (out ? 2 * DP * kPitch<DP> : 0); }
  static constexpr int ctas(int mode) { return DP == 128 ? 1 : mode == kWhole ? 2 : mode == kOutputs ? 3 : 4; }
};

// One tile's rows, n of them from p on, to shared memory, zeros behind them.  CB: bytes that every row's pieces
// allow.  Columns from D on are not touched.
template <int DP, int CB, int T>
__device__ __forceinline__ void load_tile(char* s, const bf16* p, int64_t st, int n, int D) {
  constexpr int E = CB / 2, PER = DP / E, ROWS = T / PER > 0 ? T / PER : 1;
  if constexpr (CB == 16) {
    const int row = threadIdx.x / PER, col = threadIdx.x % PER * E;
    if (col >= D) return;
    uint32_t d = shared_at(s) + row * kPitch<DP> + col * 2;
    const char* src = reinterpret_cast<const char*>(p + row * st + col);
    const int64_t step = ROWS * st * 2;
    if (n == kAttnChunk) {
#pragma unroll
      for (int m = 0; m < kAttnChunk / ROWS; ++m, src += step)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + m * ROWS * kPitch<DP>), "l"(src) : "memory");
    } else {
#pragma unroll
      for (int m = 0; m < kAttnChunk / ROWS; ++m, src += step) {
        const bool in = row + m * ROWS < n;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + m * ROWS * kPitch<DP>),
                     "l"(in ? src : reinterpret_cast<const char*>(p)), "r"(in ? 16 : 0) : "memory");
      }
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < kAttnChunk * PER; i += T) {
      const int row = i / PER, col = i % PER * E;
      if (col >= D) continue;
      char* dst = s + row * kPitch<DP> + col * 2;
      const bf16* src = p + (row < n ? row * st + col : 0);
      if constexpr (CB == 2) {
        *reinterpret_cast<bf16*>(dst) = row < n ? *src : __float2bfloat16(0.f);
      } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(shared_at(dst)), "l"(src), "r"(row < n ? 4 : 0) : "memory");
      }
    }
  }
}

template <int DP, int MODE, int CB>
__global__ void __launch_bounds__(AttnShape<DP>::kThreads, AttnShape<DP>::ctas(MODE)) attn_mma_kernel(const __grid_constant__ AttnParams p) {
  using Sh = AttnShape<DP>;
  constexpr bool OUT = MODE != kSums, EXACT = MODE != kOutputs;
  constexpr int T = Sh::kThreads, KD = DP / 16, SN = Sh::kStateCols / 8, ON = Sh::kOutCols / 8, PT = kPitch<DP>;
  constexpr int SPLITS = EXACT ? 3 : 2, STAGE = Sh::tiles(OUT) * Sh::kTile;
  extern __shared__ uint4 smem16[];
  __shared__ float pw[kAttnChunk + 1];
  // in(i) si and up(j) su of a whole chunk; a short one of n tokens reads the one that counts from the chunk's
  // end 64 - n further on
  __shared__ float entry[2 * kAttnChunk], update[2 * kAttnChunk];
  char* tiles = reinterpret_cast<char*>(smem16);
  char* rbuf = tiles + 2 * STAGE;
  const AttnPass& a = p.pass[blockIdx.z];
  const int D = p.D, back = a.backwards;
  const int64_t bh = blockIdx.x / p.nseg;
  const int seg = blockIdx.x % p.nseg;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c = lane % 4;
  const int begin = seg * p.seg, end = min(p.L, begin + p.seg);
  const int chunks = (end - begin + kAttnChunk - 1) / kAttnChunk;
  const bf16* yp = static_cast<const bf16*>(a.y.p) + b * a.y.sb + h * a.y.sh;
  const bf16* zp = static_cast<const bf16*>(a.z.p) + b * a.z.sb + h * a.z.sh;
  const bf16* xp = OUT ? static_cast<const bf16*>(a.x.p) + b * a.x.sb + h * a.x.sh : nullptr;

  let_next_start();
  const float gd = p.g[h];
  for (int i = threadIdx.x; i < 2 * kAttnChunk; i += T) {
    if (i <= kAttnChunk) pw[i] = decay_pow(gd, i);
    const bool in = i < kAttnChunk;
    entry[i] = in ? a.si * decay_pow(gd, back ? kAttnChunk - 1 - i : i + 1) : 0.f;
    update[i] = in ? a.su * decay_pow(gd, back ? i + 1 : kAttnChunk - 1 - i) : 0.f;
  }
  if (D < DP)  // columns that no copy reaches
    for (int i = threadIdx.x; i < 2 * STAGE / 16; i += T) smem16[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();

  auto chunk_at = [&](int q) { return begin + (back ? chunks - 1 - q : q) * kAttnChunk; };
  auto load = [&](int q) {
    const int t0 = chunk_at(q), n = min(kAttnChunk, end - t0);
    char* s = tiles + (q & 1) * STAGE;
    load_tile<DP, CB, T>(s, yp + (int64_t)t0 * a.y.st, a.y.st, n, D);
    load_tile<DP, CB, T>(s + Sh::kTile, zp + (int64_t)t0 * a.z.st, a.z.st, n, D);
    if (OUT) load_tile<DP, CB, T>(s + 2 * Sh::kTile, xp + (int64_t)t0 * a.x.st, a.x.st, n, D);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  load(0);
  // the tensors were there before the sums' kernel began; the states come from the kernel before this one
  if (OUT && p.nseg > 1) wait_for_previous();

  // the warp's part of the state: rows sr + g (+ 8), columns sc + 8 n + 2 c (+ 1)
  const int sr = DP == 32 ? (warp & 1) * 16 : warp * 16, sc = DP == 32 ? (warp >> 1) * 16 : 0;
  // its part of the outputs: tokens 16 r + g (+ 8), columns oc + ...  Strips go round with the CTA, since the
  // lower ones have more tiles on their side of the diagonal and a warp's number decides its sub-partition
  const int r = (warp + blockIdx.x) % 4, oc = DP == 128 ? (warp >> 2) * 64 : 0;
  float R[SN][4];
  const float* state = OUT ? entering(p, a, bh, seg) : nullptr;
  auto keep_copy = [&](int q) {  // bf16(R) for the next chunk's product
    char* rb = rbuf + (q & 1) * DP * PT + (sr + g) * PT + sc * 2 + c * 4;
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) *reinterpret_cast<uint32_t*>(rb + e * 8 * PT + n * 16) = pack2(R[n][2 * e], R[n][2 * e + 1]);
  };
#pragma unroll
  for (int n = 0; n < SN; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = sr + g + 8 * (e >> 1), col = sc + 8 * n + 2 * c + (e & 1);
      R[n][e] = OUT && state && row < D && col < D ? (a.transposed ? state[col * D + row] : state[row * D + col]) : 0.f;
    }
  // factors of P: on the diagonal's two tiles every element has its own; elsewhere decay^|i - j| is a power that
  // a tile shares times one of four (both at most 1: no power of a strong decay overflows)
  float near4[4], diag[8];
  if (OUT) {
    keep_copy(0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = g + 8 * (e >> 1), col = 2 * c + (e & 1);
      near4[e] = a.sa * pw[back ? 15 + col - row : row + 7 - col];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int d = back ? 8 * m + col - row : row - col - 8 * m;
        diag[m * 4 + e] = d >= 0 ? a.sa * pw[d] : 0.f;
      }
    }
  }
  const float* far = pw + (back ? -16 * r - 15 : 16 * r - 7);
  // one chunk: few products, whose roundings would not average out in the outputs, so P is split as well
  const bool fine = p.L <= kAttnChunk;

  // whether the weighted tokens' third part counts
  const bool third = EXACT && a.to && (OUT || decay_pow(gd, back ? begin : p.L - end) > 0x1p-8f);

  // a lane's address of four 8 x 8 blocks: rows first (la), or columns first (lb)
  const uint32_t la = (lane % 8 + 8 * ((lane / 8) % 2)) * PT + lane / 16 * 16;
  const uint32_t lb = (lane % 8 + 8 * (lane / 16)) * PT + (lane / 8) % 2 * 16;
  const uint32_t tiles_at = shared_at(tiles), rbuf_at = shared_at(rbuf) + la + oc * 2;

  uint64_t odd[2] = {0, 0};  // not finite where one of the thread's outputs is not

  for (int q = 0; q < chunks; ++q) {
    const int t0 = chunk_at(q), n_rows = min(kAttnChunk, end - t0), shift = kAttnChunk - n_rows;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // this chunk's tiles and bf16(R) are there; the other tiles and copy are no longer read
    if (q + 1 < chunks) load(q + 1);
    char* stage = tiles + (q & 1) * STAGE;
    const uint32_t Y = tiles_at + (q & 1) * STAGE, Z = Y + Sh::kTile, X = Z + Sh::kTile;
    float O[OUT ? ON : 1][4];
    uint32_t x[OUT ? KD : 1][4];
    if constexpr (OUT) {
      const uint32_t Rb = rbuf_at + (q & 1) * DP * PT, Xa = X + 16 * r * PT + la;
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        ldm4(x[k], Xa + k * 32);
#pragma unroll
        for (int n = 0; n < ON; n += 2) {
          uint32_t w[4];
          ldm4t(w, Rb + 16 * k * PT + n * 16);
          if (k == 0) {
            mma0(O[n], x[k], w[0], w[1]);
            mma0(O[n + 1], x[k], w[2], w[3]);
          } else {
            mma(O[n], x[k], w[0], w[1]);
            mma(O[n + 1], x[k], w[2], w[3]);
          }
        }
      }
      const float* in = entry + 16 * r + g + (back ? shift : 0);
      const float f0 = in[0], f1 = in[8];
#pragma unroll
      for (int n = 0; n < ON; ++n) {
        scale2(O[n][0], O[n][1], f0, f0);
        scale2(O[n][2], O[n][3], f1, f1);
      }
    }
    // the state decays over the chunk; where it is exact a chunk's products are added up apart
    const float keep = pw[n_rows];
    float U[EXACT ? SN : 1][4];
#pragma unroll
    for (int n = 0; n < SN; ++n) {
      scale2(R[n][0], R[n][1], keep, keep);
      scale2(R[n][2], R[n][3], keep, keep);
    }
    auto& acc = first_if<!EXACT>(R, U);
    const float* up = update + 2 * c + (back ? 0 : shift);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bool mine = OUT && !(back ? s < r : s > r);
      uint32_t P[4], P2[4];
      if constexpr (OUT) {
        if (mine) {
          float S[2][4];
#pragma unroll
          for (int k = 0; k < KD; ++k) {
            uint32_t w[4];
            ldm4(w, Y + lb + 16 * s * PT + k * 32);
            if (k == 0) {
              mma0(S[0], x[k], w[0], w[1]);
              mma0(S[1], x[k], w[2], w[3]);
            } else {
              mma(S[0], x[k], w[0], w[1]);
              mma(S[1], x[k], w[2], w[3]);
            }
          }
          if (s == r) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              scale2(S[m][0], S[m][1], diag[m * 4], diag[m * 4 + 1]);
              scale2(S[m][2], S[m][3], diag[m * 4 + 2], diag[m * 4 + 3]);
            }
          } else {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const float f = back ? far[16 * s + 8 * m] : far[-16 * s - 8 * m];
              float e[4] = {near4[0], near4[1], near4[2], near4[3]};
              scale2(e[0], e[1], f, f);
              scale2(e[2], e[3], f, f);
              scale2(S[m][0], S[m][1], e[0], e[1]);
              scale2(S[m][2], S[m][3], e[2], e[3]);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) P[e] = pack2(S[e >> 1][2 * (e & 1)], S[e >> 1][2 * (e & 1) + 1]);
          if (fine) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              less2(S[e >> 1][2 * (e & 1)], S[e >> 1][2 * (e & 1) + 1], P[e]);
              P2[e] = pack2(S[e >> 1][2 * (e & 1)], S[e >> 1][2 * (e & 1) + 1]);
            }
          }
        }
      }
      uint32_t y[4], part[SPLITS][4], z[SN][2];
      ldm4t(y, Y + lb + 16 * s * PT + sr * 2);
#pragma unroll
      for (int n = 0; n < SN; n += 2) {
        uint32_t w[4];
        ldm4t(w, Z + la + 16 * s * PT + sc * 2 + n * 16);
        z[n][0] = w[0]; z[n][1] = w[1]; z[n + 1][0] = w[2]; z[n + 1][1] = w[3];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // y[0], y[1]: tokens 2 c, 2 c + 1 of the 16; y[2], y[3]: 8 further
        float lo = __uint_as_float(y[e] << 16), hi = __uint_as_float(y[e] & 0xffff0000u);
        scale2(lo, hi, up[16 * s + 4 * (e & 2)], up[16 * s + 4 * (e & 2) + 1]);
#pragma unroll
        for (int k = 0; k < SPLITS; ++k) {
          if (k == 2 && !third) break;
          part[k][e] = pack2(lo, hi);
          if (k + 1 < SPLITS) less2(lo, hi, part[k][e]);
        }
      }
#pragma unroll
      for (int k = 0; k < SPLITS; ++k) {
        if (k == 2 && !third) break;
#pragma unroll
        for (int n = 0; n < SN; ++n) {
          if (EXACT && s == 0 && k == 0) mma0(acc[n], part[k], z[n][0], z[n][1]);
          else mma(acc[n], part[k], z[n][0], z[n][1]);
        }
      }
      if constexpr (OUT) {
        if (mine) {
#pragma unroll
          for (int n = 0; n < ON; n += 2) {
            uint32_t w[4];
            if constexpr (DP == 64) {  // the outputs' columns are the state's
              w[0] = z[n][0]; w[1] = z[n][1]; w[2] = z[n + 1][0]; w[3] = z[n + 1][1];
            } else {
              ldm4t(w, Z + la + 16 * s * PT + oc * 2 + n * 16);
            }
            mma(O[n], P, w[0], w[1]);
            mma(O[n + 1], P, w[2], w[3]);
            if (fine) {
              mma(O[n], P2, w[0], w[1]);
              mma(O[n + 1], P2, w[2], w[3]);
            }
          }
        }
      }
    }
    if constexpr (EXACT) {
#pragma unroll
      for (int n = 0; n < SN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) R[n][e] += U[n][e];
    }
    if constexpr (OUT) {
#pragma unroll
      for (int n = 0; n < ON; ++n) fma2(odd[n & 1], pair_bits(O[n][0], O[n][1]), pair_bits(O[n][2], O[n][3]));
      if (q + 1 < chunks) keep_copy(q + 1);
      bf16* out = static_cast<bf16*>(const_cast<void*>(a.out.p)) + b * a.out.sb + h * a.out.sh + (int64_t)t0 * a.out.st;
      // through the strip's own rows of X, which no other warp reads (wide heads: the strip's second warp)
      char* Xs = stage + 2 * Sh::kTile + 16 * r * PT + oc * 2;
      if constexpr (DP == 128) asm volatile("bar.sync %0, 64;" ::"r"(1 + r) : "memory");
      else __syncwarp();
#pragma unroll
      for (int n = 0; n < ON; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<uint32_t*>(Xs + (g + 8 * e) * PT + n * 16 + c * 4) = pack2(O[n][2 * e], O[n][2 * e + 1]);
      __syncwarp();
      // X's columns from D on become zeros again: an output there is infinity times zero where a token is not finite,
      // and would meet every token of the chunk that takes these tiles next
      if (a.out_vec) {
        const int col = lane % ON * 8;
        if (oc + col < D) {
#pragma unroll
          for (int m = 0; m < ON / 2; ++m) {
            const int row = lane / ON + m * (32 / ON);
            if (16 * r + row < n_rows)
              stg16(out + (16 * r + row) * a.out.st + oc + col, *reinterpret_cast<const uint4*>(Xs + row * PT + col * 2));
          }
        } else {
          for (int row = lane / ON; row < 16; row += 32 / ON) *reinterpret_cast<uint4*>(Xs + row * PT + col * 2) = make_uint4(0, 0, 0, 0);
        }
      } else {
        for (int i = lane; i < 16 * 8 * ON; i += 32) {
          const int row = i / (8 * ON), col = i % (8 * ON);
          bf16* at = reinterpret_cast<bf16*>(Xs + row * PT + col * 2);
          if (oc + col >= D) *at = __float2bfloat16(0.f);
          else if (16 * r + row < n_rows) out[(16 * r + row) * a.out.st + oc + col] = *at;
        }
      }
    }
  }
  float* const to = !EXACT ? nullptr : !OUT ? a.states + (bh * p.nseg + seg) * D * D : a.to ? a.to + bh * D * D : nullptr;
  auto leave = [&] {  // a segment's own sum, or the state behind a sequence of one segment
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = sr + g + 8 * (e >> 1), col = sc + 8 * n + 2 * c + (e & 1);
        if (row < D && col < D) to[row * D + col] = R[n][e];
      }
  };
  const bool later = OUT && a.to == a.from;  // it takes the place of the one before the sequence, which may be read again
  if (EXACT && to && !later) leave();
  if constexpr (OUT) {
    if (!__syncthreads_or(!all_finite(odd[0]) || !all_finite(odd[1]))) {
      if (EXACT && to && later) leave();
      return;
    }
    float* const M = reinterpret_cast<float*>(smem16);
    state_for_recurrence(p, a, bh, seg, M);
    __syncthreads();
    if (EXACT && to && later) leave();
    by_recurrence<bf16>(p, a, bh, seg, M);
  }
}

// bytes that every head's row of a tensor allows to copy at once: 16, 4 or 2
static int bytes_at_once(const AttnView& v, int D) {
  const int64_t at = (int64_t)reinterpret_cast<uintptr_t>(v.p) | v.sb * 2 | v.st * 2 | v.sh * 2 | D * 2;
  return at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : 2;
}

template <int DP, int MODE, int CB>
static int launch(const AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  using Sh = AttnShape<DP>;
  constexpr int smem = Sh::smem(MODE != kSums);
  static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is set
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    cudaFuncSetAttribute(attn_mma_kernel<DP, MODE, CB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const dim3 grid((unsigned)(bh * p.nseg), 1, passes);
  if (MODE == kOutputs && p.nseg > 1) launch_dependent(attn_mma_kernel<DP, MODE, CB>, grid, Sh::kThreads, smem, s, p);
  else attn_mma_kernel<DP, MODE, CB><<<grid, Sh::kThreads, smem, s>>>(p);
  return launch_status(MODE == kSums ? "attn_mma_kernel (sums)" : "attn_mma_kernel");
}

template <int MODE>
static int run(AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  int cb = 16;
  for (int i = 0; i < passes; ++i) {
    AttnPass& a = p.pass[i];
    cb = min(cb, min(bytes_at_once(a.y, p.D), bytes_at_once(a.z, p.D)));
    if (MODE != kSums) cb = min(cb, bytes_at_once(a.x, p.D));
    a.out_vec = MODE != kSums && bytes_at_once(a.out, p.D) == 16;
  }
  if (MODE == kOutputs && p.wide && cb == 16) {
    int status = 0;
    if (attn_out_tc(p, bh, passes, s, &status)) return status;
  }
  auto sized = [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    return cb == 16 ? launch<DP, MODE, 16>(p, bh, passes, s)
           : cb == 4 ? launch<DP, MODE, 4>(p, bh, passes, s) : launch<DP, MODE, 2>(p, bh, passes, s);
  };
  return p.D <= 32   ? sized(std::integral_constant<int, 32>())
         : p.D <= 64 ? sized(std::integral_constant<int, 64>()) : sized(std::integral_constant<int, 128>());
}

int attn_sums_bf16(AttnParams& p, int64_t bh, cudaStream_t s) { return run<kSums>(p, bh, 1, s); }
int attn_out_bf16(AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  return p.nseg == 1 && p.pass[0].to ? run<kWhole>(p, bh, passes, s) : run<kOutputs>(p, bh, passes, s);
}

}  // namespace hdc
