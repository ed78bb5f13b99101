// Outputs of decayed linear attention of bf16 tensors, heads of 33 to 64, on the tcgen05 tensor cores.
//
// A CTA of 256 threads walks the 128-token chunks of one segment of one batch and head, two CTAs per SM.  Per chunk
//   S = X Y' (128 x 128),  O1 = X R                      while the threads weight Y
//   U = [up Y hi | up Y lo]' Z                           while they make P; hi and lo, the two bf16 parts of the
//                                                        weighted tokens, give U's lanes 0-63 and 64-127
//   P = decay * S, rounded to bf16 in tensor memory      row i of a thread pair, 64 columns each
//   O2 = P Z
//   o = in(i) O1 + O2,  R <- e^n R + U hi + U lo         the state stays in the registers of half the threads
// and the next chunk's X and Y are loaded once S is done, Z once O2 and U are.  Roundings as in
// decay_attn_bf16.cu, whose m16n8k16 products (512 multiply-adds per clock and SM) bound the same work at 52 us for
// 32768 x 12 heads of 64.  Measured there 62 us (63), and 215 us (247) for the three passes of the gradient at 8 x 4096 x
// 16 heads; bytes 31 and 72 us.  Bound by a chunk's chain of dependent steps, 10 500 cycles with two CTAs on an SM (the
// tensor pipe is busy 17%): weighting Y 1200, P 1800, O2's eight products 1200, the rest read-outs, barriers and loads.
//
// Tensor memory, 256 columns: S in [0, 128); P, packed, over the first half of each thread pair's own 64 columns
// (piece k of 16 tokens comes to columns that pieces up to k have left); O1 and then O2 in [128, 192); U in [192, 256).
#include <atomic>

#include "decay_attn.cuh"
#include "tc.cuh"
#include "vec.cuh"

namespace hdc {

constexpr int kTcTokens = 128, kTcThreads = 256;
constexpr int kTcTile = kTcTokens * 128;  // bytes of a tile: rows of 64 values, 128-byte swizzle
constexpr int kTcSmem = 5 * kTcTile + 8192 + 1024;
constexpr int kTcCode = 81;  // hdc_device_error: a product that did not complete

// x, y and z of each pass as [B][L][H][D]: a chunk's tile is a box of 128 tokens and 64 values; tokens behind the
// sequence and values behind the head are zeros.
struct alignas(64) TcMaps {
  CUtensorMap m[3][3];
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) { return f2_to_bf2(f2_make(lo, hi)); }

__global__ void __launch_bounds__(kTcThreads, 2) attn_tc_kernel(const __grid_constant__ AttnParams p,
                                                                const __grid_constant__ TcMaps maps) {
  extern __shared__ uint8_t raw[];
  // products: S and O1; O2; U.  Loads: X and Y; Z
  __shared__ __align__(8) uint64_t bars[5];
  __shared__ uint32_t s_tmem;
  __shared__ int s_late, s_odd;  // a wait has run out; an output is not finite
  // powers of the decay; in(i) si and up(j) su of a whole chunk (a short one of n tokens reads the one that counts
  // from the chunk's end 128 - n further on); sa e^|i - j| at 127 + (j - i), zeros on the masked side
  __shared__ float pw[kTcTokens + 1], entry[2 * kTcTokens], update[2 * kTcTokens], apart[2 * kTcTokens];
  const uint32_t raw_at = smem_u32(raw), X = (raw_at + 1023) & ~1023u;
  const uint32_t Y = X + kTcTile, Z = Y + kTcTile, KH = Z + kTcTile, KL = KH + kTcTile, SR = KL + kTcTile;
  uint8_t* const tiles = raw + (X - raw_at);
  const AttnPass& a = p.pass[blockIdx.z];
  const int D = p.D, back = a.backwards;
  const int64_t bh = blockIdx.x / p.nseg;
  const int seg = blockIdx.x % p.nseg;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quarter = warp & 3, half = warp >> 2;
  const int row = 32 * quarter + lane;  // the thread's row of a chunk and lane of tensor memory
  // products and loads are issued by a thread whose part of P is all behind the causal mask
  const bool issues = threadIdx.x == (back ? 3 * 32 : 4 * 32);
  const int begin = seg * p.seg, end = min(p.L, begin + p.seg);
  const int chunks = (end - begin + kTcTokens - 1) / kTcTokens;
  auto* const op = static_cast<__nv_bfloat16*>(const_cast<void*>(a.out.p)) + b * a.out.sb + h * a.out.sh;

  let_next_start();
  if (warp == 0) {
    tmem_alloc(&s_tmem, 256);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 5; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
    s_late = s_odd = 0;
  }
  const float gd = p.g[h];
  for (int i = threadIdx.x; i < 2 * kTcTokens; i += kTcThreads) {
    if (i <= kTcTokens) pw[i] = decay_pow(gd, i);
    const bool in = i < kTcTokens;
    entry[i] = in ? a.si * decay_pow(gd, back ? kTcTokens - 1 - i : i + 1) : 0.f;
    update[i] = in ? a.su * decay_pow(gd, back ? i + 1 : kTcTokens - 1 - i) : 0.f;
    const int d = back ? i - (kTcTokens - 1) : kTcTokens - 1 - i;
    apart[i] = d >= 0 ? a.sa * decay_pow(gd, d) : 0.f;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem, mine = tmem + ((uint32_t)(32 * quarter) << 16);

  auto chunk_at = [&](int q) { return begin + (back ? chunks - 1 - q : q) * kTcTokens; };
  const CUtensorMap* const map = maps.m[blockIdx.z];
  auto load_xy = [&](int q) {  // one thread; so is load_z
    mbar_expect_tx(&bars[3], 2 * kTcTile);
    tma_load_4d(X, map, 0, h, chunk_at(q), b, &bars[3]);
    tma_load_4d(Y, map + 1, 0, h, chunk_at(q), b, &bars[3]);
  };
  auto load_z = [&](int q) {
    mbar_expect_tx(&bars[4], kTcTile);
    tma_load_4d(Z, map + 2, 0, h, chunk_at(q), b, &bars[4]);
  };
  if (issues) {
    load_xy(0);
    load_z(0);
  }
  // the tensors were there before the sums' kernel began; the states come from the kernel before this one
  wait_for_previous();

  // quarters 0 and 1: row `row` of the state, columns 32 half + [0, 32)
  float R[32];
  const float* state = a.states + (bh * p.nseg + seg) * D * D;
  auto keep_copy = [&] {  // bf16(R) for the next chunk's product: rows of 64 values, the columns side by side
    if (quarter >= 2) return;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint4 v;
      v.x = pack_bf16(R[8 * c], R[8 * c + 1]); v.y = pack_bf16(R[8 * c + 2], R[8 * c + 3]);
      v.z = pack_bf16(R[8 * c + 4], R[8 * c + 5]); v.w = pack_bf16(R[8 * c + 6], R[8 * c + 7]);
      *reinterpret_cast<uint4*>(tiles + 5 * kTcTile + sw128_chunk(row, 4 * half + c)) = v;
    }
    fence_proxy_async_smem();
  };
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int col = 32 * half + i;
    R[i] = quarter < 2 && row < D && col < D ? (a.transposed ? state[col * D + row] : state[row * D + col]) : 0.f;
  }
  keep_copy();

  int q = 0;
  for (; q < chunks; ++q) {
    const int t0 = chunk_at(q), n = min(kTcTokens, end - t0), shift = kTcTokens - n;
    const bool last = q + 1 == chunks;
    const uint32_t ph = q & 1;
    __syncthreads();
    if (s_late) break;
    if (!mbar_wait_warp(&bars[3], ph, kTcCode)) s_late = 1;
    if (issues) {
      tc_fence_after();
      constexpr uint32_t idS = idesc_bf16_f32(128, 128, false, false), idO = idesc_bf16_f32(128, 64, false, true);
      const uint64_t dX = sdesc_sw128(X, 16, 1024), dY = sdesc_sw128(Y, 16, 1024), dR = sdesc_sw128(SR, 0, 1024);
#pragma unroll
      for (int k = 0; k < 4; ++k) umma_bf16(tmem, dX + 2 * k, dY + 2 * k, idS, k > 0 ? 1u : 0u);
#pragma unroll
      for (int k = 0; k < 4; ++k) umma_bf16(tmem + 128, dX + 2 * k, dR + 128 * k, idO, k > 0 ? 1u : 0u);
      umma_commit(&bars[0]);
    }
    // the weighted tokens' two parts, for the state behind this chunk
    if (!last) {
      const float* up = update + (back ? 0 : shift);
      const int c = threadIdx.x % 8, r0 = threadIdx.x / 8;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int r = r0 + 32 * m, at = sw128_chunk(r, c);
        const uint4 v = *reinterpret_cast<const uint4*>(tiles + kTcTile + at);
        const float w = up[r];
        const uint64_t ww = f2_make(w, w);
        uint32_t in[4] = {v.x, v.y, v.z, v.w}, hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t x = f2_mul(bf2_to_f2(in[e]), ww);
          hi[e] = f2_to_bf2(x);
          lo[e] = f2_to_bf2(f2_sub(x, bf2_to_f2(hi[e])));
        }
        *reinterpret_cast<uint4*>(tiles + 3 * kTcTile + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(tiles + 4 * kTcTile + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    const int ksteps = (n + 15) / 16;
    const uint64_t dZ = sdesc_sw128(Z, 0, 1024);
    if (!last) {
      fence_proxy_async_smem();
      __syncthreads();
      if (issues) {
        if (!mbar_wait(&bars[4], ph, kTcCode)) s_late = 1;
        tc_fence_after();
        constexpr uint32_t idU = idesc_bf16_f32(128, 64, true, true);
        const uint64_t dK = sdesc_sw128(KH, kTcTile, 1024);
        for (int k = 0; k < ksteps; ++k) umma_bf16(tmem + 192, dK + 128 * k, dZ + 128 * k, idU, k > 0 ? 1u : 0u);
        umma_commit(&bars[2]);
      }
    }
    if (!mbar_wait_warp(&bars[0], ph, kTcCode)) s_late = 1;
    tc_fence_after();
    float o[32];
    tmem_ld32(mine + 128 + 32 * half, o);
    {
      const float f = entry[row + (back ? shift : 0)];
      const uint64_t ff = f2_make(f, f);
#pragma unroll
      for (int i = 0; i < 32; i += 2) f2_split(f2_mul(f2_make(o[i], o[i + 1]), ff), o[i], o[i + 1]);
    }
    // P: the warp's rows are [lo, lo + 32)
    const int lo = 32 * quarter;
    const float* by = apart + kTcTokens - 1 + 64 * half - row;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j0 = 64 * half + 16 * k;
      uint32_t pk[8];
      if (back ? j0 + 15 < lo : j0 > lo + 31) {
#pragma unroll
        for (int e = 0; e < 8; ++e) pk[e] = 0u;
      } else {
        float s[16];
        tmem_ld16(mine + 64 * half + 16 * k, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = 16 * k + 2 * e;
          pk[e] = f2_to_bf2(f2_mul(f2_make(s[2 * e], s[2 * e + 1]), f2_make(by[i], by[i + 1])));
        }
      }
      tmem_st8_async(mine + 64 * half + 8 * k, pk);
    }
    tmem_wait_st();
    tc_fence_before();
    fence_proxy_async_smem();
    __syncthreads();
    if (issues) {
      if (!mbar_wait(&bars[4], ph, kTcCode)) s_late = 1;
      tc_fence_after();
      constexpr uint32_t idO = idesc_bf16_f32(128, 64, false, true);
      for (int k = 0; k < ksteps; ++k)
        umma_bf16_ts(tmem + 128, tmem + 64 * (k >> 2) + 8 * (k & 3), dZ + 128 * k, idO, k > 0 ? 1u : 0u);
      umma_commit(&bars[1]);
      if (!last) load_xy(q + 1);  // the first group is done and Y is read
    }
    if (!mbar_wait_warp(&bars[1], ph, kTcCode)) s_late = 1;
    tc_fence_after();
    uint32_t out[16];
    {
      float o2[32];
      tmem_ld32(mine + 128 + 32 * half, o2);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        out[i] = f2_to_bf2(f2_add(f2_make(o[2 * i], o[2 * i + 1]), f2_make(o2[2 * i], o2[2 * i + 1])));
      uint64_t odd = f2_make(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 32; i += 4) odd = f2_fma(f2_make(o2[i], o2[i + 1]), f2_make(o2[i + 2], o2[i + 3]), odd);
      if (!all_finite(odd)) s_odd = 1;
    }
    if (!last) {
      if (!mbar_wait_warp(&bars[2], ph, kTcCode)) s_late = 1;
      tc_fence_after();
      if (issues) load_z(q + 1);
    }
    // the second group is done: the outputs go through the hi part's tile, U's lo part, rounded to bf16 (it is 2^-9 of
    // the hi part), through the lo part's
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<uint4*>(tiles + 3 * kTcTile + sw128_chunk(row, 4 * half + c)) =
          make_uint4(out[4 * c], out[4 * c + 1], out[4 * c + 2], out[4 * c + 3]);
    float u[32];
    if (!last) {
      tmem_ld32(mine + 192 + 32 * half, u);
      if (quarter >= 2) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<uint4*>(tiles + 4 * kTcTile + sw128_chunk(row - 64, 4 * half + c)) =
              make_uint4(pack_bf16(u[8 * c], u[8 * c + 1]), pack_bf16(u[8 * c + 2], u[8 * c + 3]),
                         pack_bf16(u[8 * c + 4], u[8 * c + 5]), pack_bf16(u[8 * c + 6], u[8 * c + 7]));
      }
    }
    tc_fence_before();
    __syncthreads();
    if (!last && quarter < 2) {
      const uint64_t keep = f2_make(pw[n], pw[n]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 v = *reinterpret_cast<const uint4*>(tiles + 4 * kTcTile + sw128_chunk(row, 4 * half + c));
        const uint32_t low[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 8 * c + 2 * e;
          f2_split(f2_fma(keep, f2_make(R[i], R[i + 1]), f2_add(f2_make(u[i], u[i + 1]), bf2_to_f2(low[e]))), R[i], R[i + 1]);
        }
      }
      keep_copy();
    }
    __nv_bfloat16* const to = op + (int64_t)t0 * a.out.st;
    if (a.out_vec) {
      const int c = threadIdx.x % 8, r0 = threadIdx.x / 8;
      if (c * 8 < D) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int r = r0 + 32 * m;
          if (r < n) stg16(to + r * a.out.st + c * 8, *reinterpret_cast<const uint4*>(tiles + 3 * kTcTile + sw128_chunk(r, c)));
        }
      }
    } else {
      for (int i = threadIdx.x; i < kTcTokens * 64; i += kTcThreads) {
        const int r = i / 64, c = i % 64;
        if (r < n && c < D) to[r * a.out.st + c] = *reinterpret_cast<const __nv_bfloat16*>(tiles + 3 * kTcTile + sw128_off(r, c));
      }
    }
  }
  __syncthreads();
  if (s_late) {  // a wait has run out: no load is left on its way when the CTA ends
    const uint32_t ph = min(q, chunks - 1) & 1;
    mbar_wait_warp(&bars[3], ph, kTcCode);
    mbar_wait_warp(&bars[4], ph, kTcCode);
  }
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 256);
  if (s_odd && !s_late) {
    float* M = reinterpret_cast<float*>(tiles);
    state_for_recurrence(p, a, bh, seg, M);
    __syncthreads();
    by_recurrence<__nv_bfloat16>(p, a, bh, seg, M);
  }
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static std::atomic<EncodeTiled> found{nullptr};
  EncodeTiled f = found.load(std::memory_order_acquire);
  if (!f) {
    void* at = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &at, cudaEnableDefault, &r) == cudaSuccess && r == cudaDriverEntryPointSuccess)
      f = reinterpret_cast<EncodeTiled>(at);
    found.store(f, std::memory_order_release);
  }
  return f;
}

// false where a tensor has no such map: heads that share memory, strides that the map does not hold
static bool encode(CUtensorMap* m, const AttnView& v, int64_t B, int64_t L, int64_t H, int64_t D) {
  const int64_t n[3] = {H, L, B}, s[3] = {v.sh, v.st, v.sb};
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)L, (cuuint64_t)B};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    if (n[i] > 1 && (s[i] < 1 || s[i] >= (int64_t(1) << 38))) return false;
    strides[i] = n[i] > 1 ? (cuuint64_t)s[i] * 2 : 128;
  }
  const cuuint32_t box[4] = {64, 1, kTcTokens, 1}, one[4] = {1, 1, 1, 1};
  const EncodeTiled f = encode_tiled();
  return f && f(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(v.p), dims, strides, box, one,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool attn_out_tc(const AttnParams& p, int64_t bh, int passes, cudaStream_t s, int* status) {
  TcMaps maps;
  for (int i = 0; i < passes; ++i) {
    const AttnPass& a = p.pass[i];
    const AttnView* v[3] = {&a.x, &a.y, &a.z};
    for (int k = 0; k < 3; ++k)
      if (!encode(&maps.m[i][k], *v[k], bh / p.H, p.L, p.H, p.D)) return false;
  }
  static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is set
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    cudaFuncSetAttribute(attn_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmem);
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  launch_dependent(attn_tc_kernel, dim3((unsigned)(bh * p.nseg), 1, passes), kTcThreads, kTcSmem, s, p, maps);
  *status = launch_status("attn_tc_kernel");
  return true;
}

}  // namespace hdc
