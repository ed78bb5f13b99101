// Decayed linear attention of bf16 tensors on the tensor cores (mma.sync m16n8k16, fp32 sums).
//
// A CTA walks the 64-token chunks of one segment of one batch and head.  The state R stays in fp32 in the
// accumulators of the warps, 16 rows each; a copy rounded to bf16 goes through shared memory to the product
// x R of the next chunk.  Per chunk and warp (16 tokens of outputs):
//   O = in(i) X R;  S = X Y' (the tiles on and below the diagonal);  P = decay * S;  O += P Z;  R = e^n R + (up Y)' Z.
// S becomes P in registers: an accumulator tile has the layout of the next product's operand.
//
// Roundings.  P and the copy of R are rounded to bf16 once, as the result is; sums and states stay fp32.  The
// weighted tokens up(j) y_j would add a third rounding to every state: they are split into bf16 parts, two where
// only outputs follow (2^-17), three in the segments' sums, from which the fp32 state that the caller gets is
// made (2^-25).  Those sums are also added up chunk by chunk outside the tensor cores, whose own sums of many
// steps lose low bits one-sidedly.
//
// Why not tcgen05: with heads of 64 a chunk's products are 64 x 64 x 64, each needed by the next within some
// hundred ns; through tensor memory every one of them costs a round trip (commit, wait, load, convert, store),
// as the slot kernels' 6 us per 256 tokens show, while here three or more CTAs per SM overlap theirs in registers.
// 136 products of m16n8k16 per chunk and warp come to 24 us for 32768 x 12 heads of 64, whose bytes take 31 us.
#include <atomic>

#include "decay_attn.cuh"

namespace hdc {

using bf16 = __nv_bfloat16;

// shared-memory tile [rows][DP] of bf16 in 16-byte units, swizzled so that eight neighbouring rows of one
// unit lie in different banks
template <int DP> __device__ __forceinline__ int unit_at(int row, int unit) {
  if constexpr (DP == 32) return row * 4 + (unit ^ ((row >> 1) & 3));
  else return row * (DP / 8) + (unit ^ (row & 7));
}

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
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_f(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_f(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// One tile's rows [t0, t0 + n) to shared memory, zeros behind them.  CB: bytes that every row's pieces allow.
template <int DP, int CB, int THREADS>
__device__ __forceinline__ void load_tile(bf16* s, const bf16* p, int64_t st, int n, int D) {
  constexpr int E = CB / 2;  // elements of a copy
  constexpr int PER = DP / E;
#pragma unroll 4
  for (int i = threadIdx.x; i < kAttnChunk * PER; i += THREADS) {
    const int r = i / PER, c = i % PER * E;
    if (c >= D) continue;
    bf16* dst = s + unit_at<DP>(r, c / 8) * 8 + c % 8;
    const bf16* src = p + (r < n ? r * st + c : 0);
    if constexpr (CB == 2) {
      *dst = r < n ? *src : __float2bfloat16(0.f);
    } else {
      const uint32_t d = shared_at(dst);
      const int bytes = r < n ? CB : 0;
      if constexpr (CB == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
    }
  }
}

template <bool FIRST, typename A, typename B> __device__ __forceinline__ auto& first_if(A& a, B& b) {
  if constexpr (FIRST) return a;
  else return b;
}

template <int DP> struct AttnShape {
  static constexpr int kWarps = DP == 128 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTile = kAttnChunk * DP;                   // elements of a tile
  static constexpr int kStateCols = DP == 32 ? 16 : DP;           // a warp's columns of the state (16 rows)
  static constexpr int kOutCols = DP == 128 ? 64 : DP;            // a warp's columns of the outputs (16 tokens)
  static constexpr int smem(bool out) { return 2 * ((out ? 3 : 2) * 2 * kTile + (out ? 2 * DP * DP : 0)); }
  static constexpr int ctas(bool out) { return DP == 128 ? 1 : out ? 3 : 4; }
};

template <int DP, bool OUT, int CB>
__global__ void __launch_bounds__(AttnShape<DP>::kThreads, AttnShape<DP>::ctas(OUT)) attn_mma_kernel(const __grid_constant__ AttnParams p) {
  using Sh = AttnShape<DP>;
  constexpr int T = Sh::kThreads, KD = DP / 16, SN = Sh::kStateCols / 8, ON = Sh::kOutCols / 8;
  constexpr int SPLITS = OUT ? 2 : 3;
  extern __shared__ uint4 smem16[];
  __shared__ float pw[kAttnChunk + 1];
  bf16* tiles = reinterpret_cast<bf16*>(smem16);
  bf16* rbuf = tiles + (OUT ? 3 : 2) * 2 * Sh::kTile;
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

  for (int i = threadIdx.x; i <= kAttnChunk; i += T) pw[i] = decay_pow(p.g[h], i);
  if (D < DP)  // columns that no copy reaches
    for (int i = threadIdx.x; i < (OUT ? 3 : 2) * 2 * Sh::kTile / 8; i += T) smem16[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();

  auto chunk_at = [&](int q) { return begin + (back ? chunks - 1 - q : q) * kAttnChunk; };
  auto load = [&](int q) {
    const int t0 = chunk_at(q), n = min(kAttnChunk, end - t0);
    bf16* s = tiles + (q & 1) * (OUT ? 3 : 2) * Sh::kTile;
    load_tile<DP, CB, T>(s, yp + (int64_t)t0 * a.y.st, a.y.st, n, D);
    load_tile<DP, CB, T>(s + Sh::kTile, zp + (int64_t)t0 * a.z.st, a.z.st, n, D);
    if (OUT) load_tile<DP, CB, T>(s + 2 * Sh::kTile, xp + (int64_t)t0 * a.x.st, a.x.st, n, D);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  load(0);

  // the warp's part of the state: rows sr + g (+ 8), columns sc + 8 n + 2 c (+ 1)
  const int sr = DP == 32 ? (warp & 1) * 16 : warp * 16, sc = DP == 32 ? (warp >> 1) * 16 : 0;
  // its part of the outputs: tokens 16 r + g (+ 8), columns oc + ...  Strips go round with the CTA, since the
  // lower ones have more tiles on their side of the diagonal and a warp's number decides its sub-partition
  const int r = (warp + blockIdx.x) % 4, oc = DP == 128 ? (warp >> 2) * 64 : 0;
  float R[SN][4];
  float* state = a.states + (bh * p.nseg + seg) * D * D;
  auto keep_copy = [&](int q) {  // bf16(R) for the next chunk's product
    bf16* rb = rbuf + (q & 1) * DP * DP;
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = sr + g + 8 * e, col = sc + 8 * n + 2 * c;
        *reinterpret_cast<uint32_t*>(rb + unit_at<DP>(row, col / 8) * 8 + col % 8) = pack2(R[n][2 * e], R[n][2 * e + 1]);
      }
  };
#pragma unroll
  for (int n = 0; n < SN; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = sr + g + 8 * (e >> 1), col = sc + 8 * n + 2 * c + (e & 1);
      R[n][e] = OUT && row < D && col < D ? (a.transposed ? state[col * D + row] : state[row * D + col]) : 0.f;
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

  // addresses of the four 8 x 8 blocks that a lane fetches: rows first (la), or columns first (lb)
  const int la_row = lane % 8 + 8 * ((lane / 8) % 2), la_unit = lane / 16;
  const int lb_row = lane % 8 + 8 * (lane / 16), lb_unit = (lane / 8) % 2;

  for (int q = 0; q < chunks; ++q) {
    const int t0 = chunk_at(q), n_rows = min(kAttnChunk, end - t0);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // this chunk's tiles and bf16(R) are there; the other tiles and copy are no longer read
    if (q + 1 < chunks) load(q + 1);
    bf16* Ys = tiles + (q & 1) * (OUT ? 3 : 2) * Sh::kTile;
    const uint32_t Y = shared_at(Ys), Z = Y + Sh::kTile * 2, X = Z + Sh::kTile * 2;
    uint32_t P[4][4];
    float O[OUT ? ON : 1][4];
    if constexpr (OUT) {
      const uint32_t Rb = shared_at(rbuf + (q & 1) * DP * DP);
#pragma unroll
      for (int n = 0; n < ON; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        uint32_t x[4];
        ldm4(x, X + unit_at<DP>(16 * r + la_row, 2 * k + la_unit) * 16);
#pragma unroll
        for (int n = 0; n < ON; n += 2) {
          uint32_t w[4];
          ldm4t(w, Rb + unit_at<DP>(16 * k + la_row, oc / 8 + n + la_unit) * 16);
          mma(O[n], x, w[0], w[1]);
          mma(O[n + 1], x, w[2], w[3]);
        }
      }
      const int i0 = 16 * r + g, i1 = i0 + 8;
      const float f0 = a.si * pw[back ? max(n_rows - 1 - i0, 0) : i0 + 1], f1 = a.si * pw[back ? max(n_rows - 1 - i1, 0) : i1 + 1];
#pragma unroll
      for (int n = 0; n < ON; ++n) { O[n][0] *= f0; O[n][1] *= f0; O[n][2] *= f1; O[n][3] *= f1; }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (back ? s < r : s > r) continue;
        float S[2][4] = {};
#pragma unroll
        for (int k = 0; k < KD; ++k) {
          uint32_t x[4], w[4];
          ldm4(x, X + unit_at<DP>(16 * r + la_row, 2 * k + la_unit) * 16);
          ldm4(w, Y + unit_at<DP>(16 * s + lb_row, 2 * k + lb_unit) * 16);
          mma(S[0], x, w[0], w[1]);
          mma(S[1], x, w[2], w[3]);
        }
        if (s == r) {
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[m][e] *= diag[m * 4 + e];
        } else {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const float far = pw[back ? 16 * (s - r) + 8 * m - 15 : 16 * (r - s) - 8 * m - 7];
#pragma unroll
            for (int e = 0; e < 4; ++e) S[m][e] *= far * near4[e];
          }
        }
        P[s][0] = pack2(S[0][0], S[0][1]);
        P[s][1] = pack2(S[0][2], S[0][3]);
        P[s][2] = pack2(S[1][0], S[1][1]);
        P[s][3] = pack2(S[1][2], S[1][3]);
      }
    }
    // the state decays over the chunk; the sums' kernel adds a chunk's products up apart
    const float keep = pw[n_rows];
    float U[OUT ? 1 : SN][4];
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        R[n][e] *= keep;
        if constexpr (!OUT) U[n][e] = 0.f;
      }
    auto& acc = first_if<OUT>(R, U);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint32_t y[4], part[SPLITS][4];
      ldm4t(y, Y + unit_at<DP>(16 * s + lb_row, sr / 8 + lb_unit) * 16);
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 16 * s + 2 * c + (e & 1) + 8 * (e >> 1);
        w[e] = a.su * pw[back ? j + 1 : max(n_rows - 1 - j, 0)];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // y[0], y[1]: tokens 2 c, 2 c + 1; y[2], y[3]: 8 further
        float lo = lo_f(y[e]) * w[e & 2], hi = hi_f(y[e]) * w[(e & 2) + 1];
#pragma unroll
        for (int k = 0; k < SPLITS; ++k) {
          part[k][e] = pack2(lo, hi);
          lo -= lo_f(part[k][e]);
          hi -= hi_f(part[k][e]);
        }
      }
      const bool mine = OUT && !(back ? s < r : s > r);
#pragma unroll
      for (int n = 0; n < SN; n += 2) {
        uint32_t w4[4];
        ldm4t(w4, Z + unit_at<DP>(16 * s + la_row, sc / 8 + n + la_unit) * 16);
#pragma unroll
        for (int k = SPLITS - 1; k >= 0; --k) {
          mma(acc[n], part[k], w4[0], w4[1]);
          mma(acc[n + 1], part[k], w4[2], w4[3]);
        }
        if constexpr (OUT && DP == 64) {  // the outputs' columns are the state's
          if (mine) {
            mma(O[n], P[s], w4[0], w4[1]);
            mma(O[n + 1], P[s], w4[2], w4[3]);
          }
        }
      }
      if constexpr (OUT && DP != 64) {
        if (mine) {
#pragma unroll
          for (int n = 0; n < ON; n += 2) {
            uint32_t w4[4];
            ldm4t(w4, Z + unit_at<DP>(16 * s + la_row, oc / 8 + n + la_unit) * 16);
            mma(O[n], P[s], w4[0], w4[1]);
            mma(O[n + 1], P[s], w4[2], w4[3]);
          }
        }
      }
    }
    if constexpr (!OUT) {
#pragma unroll
      for (int n = 0; n < SN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) R[n][e] += U[n][e];
    } else {
      keep_copy(q + 1);
      bf16* out = static_cast<bf16*>(const_cast<void*>(a.out.p)) + b * a.out.sb + h * a.out.sh + (int64_t)t0 * a.out.st;
      // through the strip's own rows of X, which no other warp reads (wide heads: the strip's second warp)
      bf16* Xs = Ys + 2 * Sh::kTile;
      if constexpr (DP == 128) asm volatile("bar.sync %0, 64;" ::"r"(1 + r) : "memory");
      else __syncwarp();
#pragma unroll
      for (int n = 0; n < ON; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<uint32_t*>(Xs + unit_at<DP>(16 * r + g + 8 * e, oc / 8 + n) * 8 + 2 * c) = pack2(O[n][2 * e], O[n][2 * e + 1]);
      __syncwarp();
      if (a.out_vec) {
#pragma unroll
        for (int i = lane; i < 16 * ON; i += 32) {
          const int row = 16 * r + i / ON, col = oc + i % ON * 8;
          if (row < n_rows && col < D)
            stg16(out + row * a.out.st + col, *reinterpret_cast<const uint4*>(Xs + unit_at<DP>(row, col / 8) * 8));
        }
      } else {
        for (int i = lane; i < 16 * 8 * ON; i += 32) {
          const int row = 16 * r + i / (8 * ON), col = oc + i % (8 * ON);
          if (row < n_rows && col < D) out[row * a.out.st + col] = Xs[unit_at<DP>(row, col / 8) * 8 + col % 8];
        }
      }
    }
  }
  if constexpr (!OUT) {
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = sr + g + 8 * (e >> 1), col = sc + 8 * n + 2 * c + (e & 1);
        if (row < D && col < D) state[row * D + col] = R[n][e];
      }
  }
}

// bytes that every head's row of a tensor allows to copy at once: 16, 4 or 2
static int bytes_at_once(const AttnView& v, int D) {
  const int64_t at = (int64_t)reinterpret_cast<uintptr_t>(v.p) | v.sb * 2 | v.st * 2 | v.sh * 2 | D * 2;
  return at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : 2;
}

template <int DP, bool OUT, int CB>
static int launch(const AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  using Sh = AttnShape<DP>;
  constexpr int smem = Sh::smem(OUT);
  static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is set
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    cudaFuncSetAttribute(attn_mma_kernel<DP, OUT, CB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  attn_mma_kernel<DP, OUT, CB><<<dim3((unsigned)(bh * p.nseg), 1, passes), Sh::kThreads, smem, s>>>(p);
  return launch_status(OUT ? "attn_mma_kernel" : "attn_mma_kernel (sums)");
}

template <bool OUT>
static int run(AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  int cb = 16;
  for (int i = 0; i < passes; ++i) {
    AttnPass& a = p.pass[i];
    cb = min(cb, min(bytes_at_once(a.y, p.D), bytes_at_once(a.z, p.D)));
    if (OUT) cb = min(cb, bytes_at_once(a.x, p.D));
    a.out_vec = OUT && bytes_at_once(a.out, p.D) == 16;
  }
  auto sized = [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    return cb == 16 ? launch<DP, OUT, 16>(p, bh, passes, s)
           : cb == 4 ? launch<DP, OUT, 4>(p, bh, passes, s) : launch<DP, OUT, 2>(p, bh, passes, s);
  };
  return p.D <= 32   ? sized(std::integral_constant<int, 32>())
         : p.D <= 64 ? sized(std::integral_constant<int, 64>()) : sized(std::integral_constant<int, 128>());
}

int attn_sums_bf16(AttnParams& p, int64_t bh, cudaStream_t s) { return run<false>(p, bh, 1, s); }
int attn_out_bf16(AttnParams& p, int64_t bh, int passes, cudaStream_t s) { return run<true>(p, bh, passes, s); }

}  // namespace hdc
