// Decayed linear attention of fp32 tensors on CUDA cores: products of tiles in shared memory, pairs of columns per
// instruction (128 multiply-adds per clock and SM; six bf16 products of mma.sync for one of fp32 would leave 85, of
// tcgen05 more than three times the CUDA cores' rate, for which there is no kernel here).
//
// 256 threads as 16 x 16; a thread has 4 rows of a chunk (tokens) and 2 G columns of the head, G = ceil(D / 32), which
// keeps the reads from shared memory below the arithmetic.  A row of the diagonal's side only goes through the
// tokens on that side; the rows of a warp are taken so that every sub-partition has the same number of them.
// Bound by the multiply-adds, D (D + 64) of them a token and pass beside the state's D^2, at 40 to 48% of the issue slots:
// a chunk's loads are waited for with nothing else in flight.  3 x 1537 x 4 heads of 96: sums 23 us, outputs 46, the
// gradient's three passes 95.
#include <atomic>
#include <type_traits>

#include "decay_attn.cuh"
#include "vec.cuh"

namespace hdc {

template <int G> struct F32Shape {
  // row pitches: X and Z; Y; R (transposed states are stored four rows apart); P
  static constexpr int kD = 32 * G, kY = kD + 4, kR = kD + 2, kP = kAttnChunk + 4;
  static constexpr int kX = kAttnChunk * (kD > kP ? kD : kP);          // X, and P in its place
  static constexpr int smem(bool out) { return 4 * ((out ? kX : 0) + kAttnChunk * (kY + kD) + kD * kR); }
  static constexpr int ctas(bool out) { return G == 4 ? 1 : G == 3 ? 2 : 3; }
};

__device__ __forceinline__ void fma2(uint64_t& s, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(s) : "l"(a), "l"(b));
}
__device__ __forceinline__ void mul2(uint64_t& s, float f) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(s) : "l"(pair_bits(f, f)));
}
__device__ __forceinline__ uint64_t two(const float* p) { return *reinterpret_cast<const uint64_t*>(p); }
__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }

// Rows [0, n) of D values from p on to shared memory, zeros behind them and in the columns from D on.
template <int KD, bool VEC>
__device__ __forceinline__ void load_rows(float* s, int pitch, const float* p, int64_t st, int n, int D) {
  constexpr int E = VEC ? 4 : 1, PER = KD / E;
#pragma unroll 8
  for (int i = threadIdx.x; i < kAttnChunk * PER; i += 256) {
    const int r = i / PER, c = i % PER * E;
    const bool in = r < n && c < D;
    if constexpr (VEC) {
      const uint4 v = ldg16_pred(in ? p + r * st + c : p, in);
      *reinterpret_cast<uint4*>(s + r * pitch + c) = v;
    } else {
      s[r * pitch + c] = in ? p[r * st + c] : 0.f;
    }
  }
}

// A state (NULL: zeros) to shared memory; zeros in the rows and columns from D on.
template <int KD, bool VEC>
__device__ __forceinline__ void load_state(float* R, int pitch, const float* state, int transposed, int D) {
  constexpr int E = VEC ? 4 : 1, PER = KD / E;
#pragma unroll 4
  for (int i = threadIdx.x; i < KD * PER; i += 256) {
    const int r = i / PER, c = i % PER * E;  // of the state in memory
    const bool in = state && r < D && c < D;
    float x[E];
    if constexpr (VEC) {
      // written by the kernel before this one: not through the read-only path
      *reinterpret_cast<float4*>(x) = in ? *reinterpret_cast<const float4*>(state + r * D + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      x[0] = in ? state[r * D + c] : 0.f;
    }
    if (transposed) {
#pragma unroll
      for (int e = 0; e < E; ++e) R[(c + e) * pitch + r] = x[e];
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) R[r * pitch + c + e] = x[e];
    }
  }
}

template <int G, bool OUT, bool VEC>
__global__ void __launch_bounds__(256, F32Shape<G>::ctas(OUT)) attn_f32_kernel(const __grid_constant__ AttnParams p) {
  using Sh = F32Shape<G>;
  constexpr int KD = Sh::kD, PY = Sh::kY, PR = Sh::kR, PP = Sh::kP;
  extern __shared__ float4 smem4[];
  float* Z = reinterpret_cast<float*>(smem4);
  float* Y = Z + kAttnChunk * KD;
  float* X = Y + kAttnChunk * PY;
  float* P = X;
  float* R = OUT ? X + Sh::kX : X;
  __shared__ float pw[kAttnChunk + 1];
  __shared__ int s_odd;  // an output is not finite
  const AttnPass& a = p.pass[blockIdx.z];
  const int D = p.D, DR = (D + 3) & ~3, back = a.backwards;
  const int64_t bh = blockIdx.x / p.nseg;
  const int seg = blockIdx.x % p.nseg;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int warp = threadIdx.x / 32, tx = threadIdx.x % 16, half = threadIdx.x / 16 % 2;
  // a warp's eight rows of the chunk: warps w and w + 4 share a sub-partition and take blocks w and 7 - w
  const int block = warp < 4 ? warp : 11 - warp, row0 = block * 8 + half * 4;
  const int begin = seg * p.seg, end = min(p.L, begin + p.seg);
  const float* xp = OUT ? static_cast<const float*>(a.x.p) + b * a.x.sb + h * a.x.sh : nullptr;
  const float* yp = static_cast<const float*>(a.y.p) + b * a.y.sb + h * a.y.sh;
  const float* zp = static_cast<const float*>(a.z.p) + b * a.z.sb + h * a.z.sh;
  const float* state = OUT ? entering(p, a, bh, seg) : nullptr;
  // the state behind the segment goes: a segment's own sum, or the state behind a sequence of one segment
  float* to = !OUT ? a.states + (bh * p.nseg + seg) * D * D : p.nseg == 1 && a.to ? a.to + bh * D * D : nullptr;
  const int chunks = (end - begin + kAttnChunk - 1) / kAttnChunk;
  let_next_start();
  if (OUT && threadIdx.x == 0) s_odd = 0;
  for (int i = threadIdx.x; i <= kAttnChunk; i += 256) pw[i] = decay_pow(p.g[h], i);
  for (int q = 0; q < chunks; ++q) {
    const int t0 = begin + (back ? chunks - 1 - q : q) * kAttnChunk, n = min(kAttnChunk, end - t0);
    load_rows<KD, VEC>(Y, PY, yp + (int64_t)t0 * a.y.st, a.y.st, n, D);
    load_rows<KD, VEC>(Z, KD, zp + (int64_t)t0 * a.z.st, a.z.st, n, D);
    if (OUT) load_rows<KD, VEC>(X, KD, xp + (int64_t)t0 * a.x.st, a.x.st, n, D);
    if (q == 0) {
      if (OUT) wait_for_previous();  // the states come from the kernel before this one
      load_state<KD, VEC>(R, PR, OUT ? state : nullptr, a.transposed, D);
    }
    __syncthreads();
    if constexpr (OUT) {
      // O = in(i) X R
      uint64_t o[4][G] = {};
      for (int d = 0; d < DR; d += 4) {
        float4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = four(X + (row0 + i) * KD + d);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint64_t w[G];
#pragma unroll
          for (int m = 0; m < G; ++m) w[m] = two(R + (d + k) * PR + tx * 2 + 32 * m);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = k == 0 ? u[i].x : k == 1 ? u[i].y : k == 2 ? u[i].z : u[i].w;
            const uint64_t xx = pair_bits(x, x);
#pragma unroll
            for (int m = 0; m < G; ++m) fma2(o[i][m], xx, w[m]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = back ? n - 1 - (row0 + i) : row0 + i + 1;
        const float f = e >= 0 ? a.si * pw[e] : 0.f;
#pragma unroll
        for (int m = 0; m < G; ++m) mul2(o[i][m], f);
      }
      // S = X Y' at columns tx + 16 j of the 16-token blocks on the rows' side of the diagonal
      float s[4][4] = {};
      const int first = back ? block / 2 : 0, last = back ? 3 : block / 2;
      for (int d = 0; d < DR; d += 4) {
        float4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = four(X + (row0 + i) * KD + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j < first || j > last) continue;
          const float4 w = four(Y + (tx + 16 * j) * PY + d);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[i][j] = fmaf(u[i].w, w.w, fmaf(u[i].z, w.z, fmaf(u[i].y, w.y, fmaf(u[i].x, w.x, s[i][j]))));
        }
      }
      __syncthreads();  // X is read: P takes its place
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j < first || j > last) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = row0 + i, c = tx + 16 * j, apart = back ? c - r : r - c;
          P[r * PP + c] = apart >= 0 ? a.sa * pw[apart] * s[i][j] : 0.f;
        }
      }
      __syncwarp();  // a warp reads its own rows
      for (int d = first * 16; d < last * 16 + 16; d += 4) {
        float4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = four(P + (row0 + i) * PP + d);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint64_t w[G];
#pragma unroll
          for (int m = 0; m < G; ++m) w[m] = two(Z + (d + k) * KD + tx * 2 + 32 * m);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = k == 0 ? u[i].x : k == 1 ? u[i].y : k == 2 ? u[i].z : u[i].w;
            const uint64_t xx = pair_bits(x, x);
#pragma unroll
            for (int m = 0; m < G; ++m) fma2(o[i][m], xx, w[m]);
          }
        }
      }
      uint64_t odd[2] = {0, 0};
#pragma unroll
      for (int m = 0; m < G; ++m) {
        fma2(odd[0], o[0][m], o[1][m]);
        fma2(odd[1], o[2][m], o[3][m]);
      }
      if (!all_finite(odd[0]) || !all_finite(odd[1])) s_odd = 1;
      float* out = static_cast<float*>(const_cast<void*>(a.out.p)) + b * a.out.sb + h * a.out.sh + (int64_t)t0 * a.out.st;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < G; ++m) {
          const int r = row0 + i, c = tx * 2 + 32 * m;
          if (r >= n || c >= D) continue;
          float* to = out + r * a.out.st + c;
          if (VEC && a.out_vec) {
            *reinterpret_cast<uint64_t*>(to) = o[i][m];
          } else {
            float v0, v1;
            bits_pair(o[i][m], v0, v1);
            to[0] = v0;
            if (c + 1 < D) to[1] = v1;
          }
        }
    }
    if (to || q + 1 < chunks) {
      // R = e^n R + sum up(j) y_j z_j': rows 2 ty + 32 k, columns 2 tx + 32 m (+ 1)
      const int ty = threadIdx.x / 16;
      uint64_t r[2 * G][G];
#pragma unroll
      for (int k = 0; k < 2 * G; ++k)
#pragma unroll
        for (int m = 0; m < G; ++m) {
          r[k][m] = two(R + (ty * 2 + 32 * (k / 2) + k % 2) * PR + tx * 2 + 32 * m);
          mul2(r[k][m], pw[n]);
        }
#pragma unroll 4
      for (int t = 0; t < n; ++t) {
        const float f = a.su * pw[back ? t + 1 : n - 1 - t];
        uint64_t w[G];
#pragma unroll
        for (int m = 0; m < G; ++m) w[m] = two(Z + t * KD + tx * 2 + 32 * m);
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const float2 y = *reinterpret_cast<const float2*>(Y + t * PY + ty * 2 + 32 * k);
          const float y0 = y.x * f, y1 = y.y * f;
          const uint64_t a0 = pair_bits(y0, y0), a1 = pair_bits(y1, y1);
#pragma unroll
          for (int m = 0; m < G; ++m) {
            fma2(r[2 * k][m], a0, w[m]);
            fma2(r[2 * k + 1][m], a1, w[m]);
          }
        }
      }
      __syncthreads();  // R, P, Y and Z are read
#pragma unroll
      for (int k = 0; k < 2 * G; ++k)
#pragma unroll
        for (int m = 0; m < G; ++m)
          *reinterpret_cast<uint64_t*>(R + (ty * 2 + 32 * (k / 2) + k % 2) * PR + tx * 2 + 32 * m) = r[k][m];
    }
  }
  __syncthreads();
  const bool redo = OUT && s_odd != 0;
  if (redo) {  // (in the place of Z and Y)
    state_for_recurrence(p, a, bh, seg, Z);
    __syncthreads();  // the state behind the sequence may take the place of the one before it
  }
  if (to)
    for (int i = threadIdx.x; i < D * D; i += 256) to[i] = R[i / D * PR + i % D];
  if (redo) by_recurrence<float>(p, a, bh, seg, Z);
}

template <int G, bool OUT, bool VEC> static int launch(const AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  constexpr int smem = F32Shape<G>::smem(OUT);
  static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is set
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    cudaFuncSetAttribute(attn_f32_kernel<G, OUT, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const dim3 grid((unsigned)(bh * p.nseg), 1, passes);
  if (OUT && p.nseg > 1) launch_dependent(attn_f32_kernel<G, OUT, VEC>, grid, 256, smem, s, p);
  else attn_f32_kernel<G, OUT, VEC><<<grid, 256, smem, s>>>(p);
  return launch_status(OUT ? "attn_f32_kernel" : "attn_f32_kernel (sums)");
}

// every head's row allows 16-byte accesses
static bool vectors(const AttnView& v, int D) {
  return (((int64_t)reinterpret_cast<uintptr_t>(v.p) | v.sb * 4 | v.st * 4 | v.sh * 4 | D * 4) & 15) == 0;
}

template <bool OUT> static int run(AttnParams& p, int64_t bh, int passes, cudaStream_t s) {
  bool vec = true;
  for (int i = 0; i < passes; ++i) {
    AttnPass& a = p.pass[i];
    // (a state's rows of D values: D * 4 bytes are looked at with the tensors')
    vec = vec && aligned16(a.states) && aligned16(a.from) && vectors(a.y, p.D) && vectors(a.z, p.D) && (!OUT || vectors(a.x, p.D));
    a.out_vec = OUT && vectors(a.out, p.D);
  }
  auto sized = [&](auto g) {
    constexpr int G = decltype(g)::value;
    return vec ? launch<G, OUT, true>(p, bh, passes, s) : launch<G, OUT, false>(p, bh, passes, s);
  };
  return p.D <= 32   ? sized(std::integral_constant<int, 1>())
         : p.D <= 64 ? sized(std::integral_constant<int, 2>())
         : p.D <= 96 ? sized(std::integral_constant<int, 3>()) : sized(std::integral_constant<int, 4>());
}

int attn_sums_f32(AttnParams& p, int64_t bh, cudaStream_t s) { return run<false>(p, bh, 1, s); }
int attn_out_f32(AttnParams& p, int64_t bh, int passes, cudaStream_t s) { return run<true>(p, bh, passes, s); }

}  // namespace hdc
