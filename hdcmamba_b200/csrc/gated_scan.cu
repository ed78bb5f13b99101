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
// Forward schedule (bound by HBM: 3 values read and 1 written per step and channel): the
// sequence is cut into tiles of 64 steps x 128 bytes of channels (64 bf16, 32 fp32).  A step is
// the map h -> a h + u, and maps compose: (P, H) then (P', H') is (P' P, P' H + H'), so each
// tile is scanned from a zero state, and the state entering it is added afterwards through P:
//   * a warp owns 8 steps of the tile, a lane one 4-byte word of channels; its a and u stay in
//     registers between the local scan and the outputs, so every input is read once;
//   * the 8 warps' maps are composed through shared memory, and the tile's map is published in
//     the workspace;
//   * the state entering the tile is composed from at most 31 published entries: the state at
//     the end of the last whole 256 tiles, the maps of the whole 16-tile spans after it, and the
//     maps of the tiles after those.  Which entries is a matter of the tile's index alone, so
//     the result does not depend on timing.
// CTAs take tiles by ticket, time-major: a tile waits only for tiles with smaller tickets,
// which running CTAs hold, so the waits end (they are bounded all the same).  An entry is one
// 64-bit word per channel, (P, H); the workspace is set to all ones before the launch, which
// no published P is, so the word is its own flag.  The next tile is in flight (cp.async)
// while one is computed.
// P < 0 marks a map that a reset has cut off from what came before (P is otherwise >= 0).
#include <type_traits>

#include "tc.cuh"

namespace hdc {

constexpr int kStateRows = 64;       // rows per tile = rows per saved state
constexpr int kWarps = 8, kRows = 8;  // warps per tile, steps per warp
constexpr int kSpan = 16;            // tiles per span, spans per chain link
#ifndef FC
#define FC 4
#endif
constexpr int kFwdCtas = FC;          // resident forward CTAs per SM
static_assert(kWarps * kRows == kStateRows, "a tile is one state interval");

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
  // tiles
  int nch;          // channel groups
  int NG;           // channel groups of all batches
  int64_t ntiles;   // NG * NT
  unsigned* ticket;  // NULL: a single tile in time, taken by block index, nothing published
  uint64_t* ent;    // [NG][NT + spans + links][CW] published entries
  int nent;         // entries per group
  int out_vec;      // the outputs' rows allow whole words
};

__device__ __forceinline__ float ld_param(const void* p, int bf16, int i) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

// softplus with the Block's threshold (hdcmamba/model.py:192), exact for small exp(x) too
__device__ __forceinline__ float softplus_acc(float x) { return x > 20.0f ? x : log1pf(expf(x)); }

// ---------------------------------------------------------------- one word of channels
// The channels of a lane: one fp32 value, or two bf16 values computed as a pair
// (fma.rn.f32x2 and friends: two fp32 operations per issued instruction).
template <int V> struct Fv { float v[V]; };
template <typename T> constexpr int kVec = 4 / sizeof(T);
template <typename T> constexpr int kCW = 32 * kVec<T>;  // channels per tile

__device__ __forceinline__ uint64_t f2_bits(const Fv<2>& a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.v[0]), "f"(a.v[1]));
  return r;
}
__device__ __forceinline__ Fv<2> bits_f2(uint64_t b) {
  Fv<2> r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.v[0]), "=f"(r.v[1]) : "l"(b));
  return r;
}
__device__ __forceinline__ Fv<1> fma(const Fv<1>& a, const Fv<1>& b, const Fv<1>& c) {
  return {{fmaf(a.v[0], b.v[0], c.v[0])}};
}
__device__ __forceinline__ Fv<1> operator*(const Fv<1>& a, const Fv<1>& b) { return {{a.v[0] * b.v[0]}}; }
__device__ __forceinline__ Fv<1> operator+(const Fv<1>& a, const Fv<1>& b) { return {{a.v[0] + b.v[0]}}; }
__device__ __forceinline__ Fv<2> fma(const Fv<2>& a, const Fv<2>& b, const Fv<2>& c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
  return bits_f2(r);
}
__device__ __forceinline__ Fv<2> operator*(const Fv<2>& a, const Fv<2>& b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return bits_f2(r);
}
__device__ __forceinline__ Fv<2> operator+(const Fv<2>& a, const Fv<2>& b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return bits_f2(r);
}
template <int V> __device__ __forceinline__ Fv<V> all(float x) {
  Fv<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = x;
  return r;
}
__device__ __forceinline__ Fv<1> word_f(uint32_t w, float) { return {{__uint_as_float(w)}}; }
__device__ __forceinline__ Fv<2> word_f(uint32_t w, __nv_bfloat16) {
  return {{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}};
}
__device__ __forceinline__ uint32_t f_word(const Fv<1>& a) { return __float_as_uint(a.v[0]); }
__device__ __forceinline__ uint32_t f_word(const Fv<2>& a) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a.v[0], a.v[1]);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// a word of dt = -inf
__device__ __forceinline__ uint32_t no_step(float) { return 0xff800000u; }
__device__ __forceinline__ uint32_t no_step(__nv_bfloat16) { return 0xff80ff80u; }
// store a word of channels c, c+1, ... (< ds); vec: the row allows the whole word
template <typename T>
__device__ __forceinline__ void st_word(T* row, int c, int ds, int vec, const Fv<kVec<T>>& v) {
  if (vec && c + kVec<T> <= ds) {
    *reinterpret_cast<uint32_t*>(row + c) = f_word(v);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (c + i < ds) row[c + i] = from_f<T>(v.v[i]);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// d = softplus(x) and a = exp(d A) for the lane's channels.
//   fp32: the library's exp and log1p.
//   bf16 inputs: softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) by the hardware's 2^x, and
//   log1p(e) = e p(e) on [0, 1] with p of degree 7, fitted here for the least relative error
//   (weighted least squares on Chebyshev points, weights iterated to equal errors: 2e-7, 3e-7
//   with fp32 evaluation; the bf16 input itself is 2^-9 off).  e p(e) keeps its relative accuracy
//   for small e, where log(1 + e) loses it.  A2 = A log2(e).
__device__ __forceinline__ void gates(const Fv<1>& x, const Fv<1>& A, const Fv<1>&, Fv<1>& d, Fv<1>& a) {
  d.v[0] = softplus_acc(x.v[0]);
  a.v[0] = expf(d.v[0] * A.v[0]);
}
__device__ __forceinline__ void gates(const Fv<2>& x, const Fv<2>&, const Fv<2>& A2, Fv<2>& d, Fv<2>& a) {
  Fv<2> e, m;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    e.v[i] = ex2(-1.4426950408889634f * fabsf(x.v[i]));
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(m.v[i]) : "f"(x.v[i]));  // NaN stays NaN
  }
#ifdef SCALARP
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float q = -0.008539206348359585f, z = e.v[i];
    q = fmaf(q, z, 0.04408962279558182f);
    q = fmaf(q, z, -0.10768169909715652f);
    q = fmaf(q, z, 0.17745240032672882f);
    q = fmaf(q, z, -0.24495463073253632f);
    q = fmaf(q, z, 0.33275479078292847f);
    q = fmaf(q, z, -0.4999740421772003f);
    q = fmaf(q, z, 0.9999998211860657f);
    d.v[i] = fmaf(q, z, m.v[i]);
  }
#else
  Fv<2> p = all<2>(-0.008539206348359585f);
  p = fma(p, e, all<2>(0.04408962279558182f));
  p = fma(p, e, all<2>(-0.10768169909715652f));
  p = fma(p, e, all<2>(0.17745240032672882f));
  p = fma(p, e, all<2>(-0.24495463073253632f));
  p = fma(p, e, all<2>(0.33275479078292847f));
  p = fma(p, e, all<2>(-0.4999740421772003f));
  p = fma(p, e, all<2>(0.9999998211860657f));
  d = fma(p, e, m);
#endif
  const Fv<2> l = d * A2;
  a.v[0] = ex2(l.v[0]);
  a.v[1] = ex2(l.v[1]);
}

// ---------------------------------------------------------------- maps h -> P h + H
template <int V> struct Map { Fv<V> P, H; };
template <int V> __device__ __forceinline__ Map<V> identity_map() { return {all<V>(1.f), all<V>(0.f)}; }
// m applied to a state (RESET: maps may be cut off)
template <bool RESET, int V> __device__ __forceinline__ Fv<V> apply(const Map<V>& m, const Fv<V>& h) {
  Fv<V> r = fma(m.P, h, m.H);
  if (RESET) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = m.P.v[i] < 0.f ? m.H.v[i] : r.v[i];
  }
  return r;
}
// first m, then n
template <bool RESET, int V> __device__ __forceinline__ Map<V> then(const Map<V>& m, const Map<V>& n) {
  Map<V> r;
  r.H = apply<RESET>(n, m.H);
  r.P = m.P * n.P;
  if (RESET) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.P.v[i] = (m.P.v[i] < 0.f || n.P.v[i] < 0.f) ? -1.f : r.P.v[i];
  }
  return r;
}
// a lane's map in shared memory: 8 bytes per channel
template <int V> __device__ __forceinline__ void st_map(char* p, int lane, const Map<V>& m) {
  float* f = reinterpret_cast<float*>(p) + lane * 2 * V;
  if constexpr (V == 2) *reinterpret_cast<float4*>(f) = make_float4(m.P.v[0], m.P.v[1], m.H.v[0], m.H.v[1]);
  else *reinterpret_cast<float2*>(f) = make_float2(m.P.v[0], m.H.v[0]);
}
template <int V> __device__ __forceinline__ Map<V> ld_map(const char* p, int lane) {
  const float* f = reinterpret_cast<const float*>(p) + lane * 2 * V;
  if constexpr (V == 2) {
    const float4 q = *reinterpret_cast<const float4*>(f);
    return {{{q.x, q.y}}, {{q.z, q.w}}};
  } else {
    const float2 q = *reinterpret_cast<const float2*>(f);
    return {{{q.x}}, {{q.y}}};
  }
}

// ---------------------------------------------------------------- published entries
constexpr uint32_t kUnset = 0xffffffffu;  // P of a word that is not published
template <int V> __device__ __forceinline__ void publish(uint64_t* e, int lane, const Map<V>& m) {
  uint64_t w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    uint32_t P = __float_as_uint(m.P.v[i]);
    if (P == kUnset) P = 0x7fffffffu;  // a NaN stays one
    w[i] = ((uint64_t)__float_as_uint(m.H.v[i]) << 32) | P;
  }
  if constexpr (V == 2)
    asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(e + lane * 2), "l"(w[0]), "l"(w[1]) : "memory");
  else asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(e + lane), "l"(w[0]) : "memory");
}
__device__ __forceinline__ void ld_entry(const uint64_t* e, uint64_t (&w)[1]) {
  asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(w[0]) : "l"(e) : "memory");
}
__device__ __forceinline__ void ld_entry(const uint64_t* e, uint64_t (&w)[2]) {
  asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(w[0]), "=l"(w[1]) : "l"(e) : "memory");
}
// Compose n in 1..4 neighbouring entries, waited for (some 2 s, then error 61; what is missing
// then counts as zeros).  e: entry 0 of them, ch: the lane's first channel.  While an entry is
// missing, one word of each is polled, not the whole entries.
constexpr long long kWaitCycles = 4000000000ll;
template <bool RESET, int V> __device__ __forceinline__ Map<V> take(const uint64_t* e, int ch, int n, int lane) {
  uint64_t w[4][V];
  long long t0 = 0;
  while (true) {
    bool ok = true;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) ld_entry(e + (int64_t)k * 32 * V + ch, w[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) ok = ok && (k >= n || (uint32_t)w[k][i] != kUnset);
    if (__all_sync(0xffffffffu, ok)) break;
    if (t0 == 0) t0 = clock64();
    bool late = false;
    if (lane < n) {
      uint64_t one[1];
      do {
        __nanosleep(32);
        ld_entry(e + (int64_t)lane * 32 * V, one);
        late = clock64() - t0 > kWaitCycles;
      } while ((uint32_t)one[0] == kUnset && !late);
    }
    if (__any_sync(0xffffffffu, late)) {
      if (lane == 0) atomicCAS(&g_dev_error, 0, 61);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if ((uint32_t)w[k][i] == kUnset) w[k][i] = 0;
      break;
    }
  }
  Map<V> m;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < n) {
      Map<V> q;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        q.P.v[i] = __uint_as_float((uint32_t)w[k][i]);
        q.H.v[i] = __uint_as_float((uint32_t)(w[k][i] >> 32));
      }
      m = k == 0 ? q : then<RESET>(m, q);
    }
  return m;
}
// Entries of a group: tiles, then spans of 16 tiles, then links of 16 spans (P unused, H the
// state itself).
__device__ __forceinline__ int span_at(int NT, int k) { return NT + k; }
__device__ __forceinline__ int link_at(int NT, int k) { return NT + (NT + kSpan - 1) / kSpan + k; }

// ---------------------------------------------------------------- staging
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool ok, std::integral_constant<int, 16>) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool ok, std::integral_constant<int, 4>) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Copies of one warp's 8 rows of 128 bytes of a tile, rows >= nv and channels >= nc as zeros.
// CB: bytes per copy (16 or 4, as the rows allow), or 0: element by element, not asynchronous.
template <typename T, int CB> struct Rows {
  static constexpr int kPer = CB ? 128 / CB : 32, kAt = 32 / kPer, kN = kRows / kAt;
  uint32_t dst;   // the lane's place in a region
  int r0, x;      // its first row and first byte of the rows
  __device__ explicit Rows(int lane) : r0(lane / kPer), x(lane % kPer * (CB ? CB : 4)) { dst = r0 * 128 + x; }
  // tile: the tile's first element; row0: the warp's first row in it; st: row stride (elements);
  // `arrays` consecutive regions, their sources `apart` elements from each other
  template <int arrays>
  __device__ __forceinline__ void copy(char* region, const T* tile, int row0, int64_t st, int64_t apart, int nv,
                                       int nc) const {
    if constexpr (CB == 0) {
      const int c = x / (int)sizeof(T);
#pragma unroll
      for (int k = 0; k < arrays; ++k)
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i)
            reinterpret_cast<T*>(region + (k * kRows + r) * 128)[c + i] =
                r < nv && c + i < nc ? tile[k * apart + (row0 + r) * st + c + i] : from_f<T>(0.f);
    } else {
      const uint32_t d = smem_u32(region) + dst;
      const bool in = x < nc * (int)sizeof(T);
      const char* src[kN];
      bool ok[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        ok[i] = in && r0 + i * kAt < nv;
        src[i] = reinterpret_cast<const char*>(tile) + (ok[i] ? (row0 + r0 + i * kAt) * st * (int64_t)sizeof(T) + x : 0);
      }
#pragma unroll
      for (int k = 0; k < arrays; ++k)
#pragma unroll
        for (int i = 0; i < kN; ++i)
          cp_async(d + (k * kRows + i * kAt) * 128, src[i] + k * apart * (int64_t)sizeof(T), ok[i],
                   std::integral_constant<int, CB>());
    }
  }
};

// A tile as broadcast through shared memory: index in time, group, batch, first channel; q < 0: none
using Tile = int4;
template <typename T> __device__ __forceinline__ Tile tile_of(const ScanParams& p, int64_t id) {
  if (id >= p.ntiles) return make_int4(-1, 0, 0, 0);
  const unsigned q = (unsigned)id / (unsigned)p.NG, g = (unsigned)id - q * p.NG, b = g / (unsigned)p.nch;
  return make_int4((int)q, (int)g, (int)b, (int)(g - b * p.nch) * kCW<T>);
}
__device__ __forceinline__ int64_t next_tile(const ScanParams& p, int64_t last) {
  if (!p.ticket) return last + gridDim.x;
  return (int64_t)(unsigned)(atomicAdd(p.ticket, 1u) + 1u);  // the counter starts at all ones
}

template <typename T, bool RESET, int CB>
__global__ void __launch_bounds__(kWarps * 32, kFwdCtas) gated_scan_fwd_kernel(const __grid_constant__ ScanParams p) {
  constexpr int V = kVec<T>, CW = kCW<T>, kRegion = 3 * kRows * 128;
  extern __shared__ __align__(128) char raw[];  // [2][warp][dt, x, b][row][128 bytes]
  __shared__ __align__(16) float s_A[2][CW];
  __shared__ Tile s_next[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cl = lane * V;  // the lane's first channel of the tile
  const Rows<T, CB> rows(lane);
  int64_t id = 0;  // thread 0's

  uint32_t rb = 0;  // the staged tile's reset flag of step `lane` of the warp
  auto stage = [&](const Tile& t, int s) {
    const int t0 = t.x * kStateRows, nv = p.L - t0 - warp * kRows, nc = p.ds - t.w;
    const T* tile = static_cast<const T*>(p.projs) + t.z * p.psb + t0 * p.pst + t.w;
    rows.template copy<3>(raw + (s * kWarps + warp) * kRegion, tile, warp * kRows, p.pst, p.ds, nv, nc);
    cp_commit();
    if (RESET) rb = lane < min(nv, kRows) ? p.reset[(int64_t)t.z * p.L + t0 + warp * kRows + lane] : 0;
    if (warp == 3) {
#pragma unroll
      for (int i = 0; i < V; ++i) s_A[s][cl + i] = cl + i < nc ? -expf(ld_param(p.A_log, p.a_bf16, t.w + cl + i)) : 0.f;
    }
  };

  if (threadIdx.x == 0) {
    id = p.ticket ? next_tile(p, 0) : blockIdx.x;
    s_next[0] = tile_of<T>(p, id);
  }
  __syncthreads();
  Tile t = s_next[0];
  if (t.x >= 0) stage(t, 0);
  __syncthreads();
  bool first = true;
  for (int s = 0; t.x >= 0; s ^= 1) {
    // The next ticket, early enough to stage its tile below.  The first time only after the loads:
    // a CTA that starts early would else take two neighbouring tiles, and the tiles after
    // the second one would wait until it is done with the first.
    if (first) cp_wait_all();
    first = false;
    if (threadIdx.x == 0) {
      id = next_tile(p, id);
      s_next[s ^ 1] = tile_of<T>(p, id);
    }
    char* buf = raw + s * kWarps * kRegion;
    char* mine = buf + warp * kRegion;
    const int t0 = t.x * kStateRows + warp * kRows, nv = p.L - t0, nc = p.ds - t.w;
    const uint32_t cut = RESET ? __ballot_sync(0xffffffffu, rb != 0) : 0;
    Fv<V> A;
#pragma unroll
    for (int i = 0; i < V; ++i) A.v[i] = s_A[s][cl + i];
    const Fv<V> A2 = A * all<V>(1.4426950408889634f);
    cp_wait_all();
    __syncwarp();
    if (nv < kRows) {  // steps past the end: dt = -inf (and x = b = 0) is the identity, a = 1, u = 0
      for (int r = max(nv, 0); r < kRows; ++r) reinterpret_cast<uint32_t*>(mine + r * 128)[lane] = no_step(T());
    }

    // local scan of the warp's steps from a zero state
    Fv<V> a[kRows], u[kRows];
    Map<V> m = identity_map<V>();
    const uint32_t* w = reinterpret_cast<const uint32_t*>(mine) + lane;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const Fv<V> dt = word_f(w[r * 32], T()), x = word_f(w[(kRows + r) * 32], T());
      const Fv<V> b = word_f(w[(2 * kRows + r) * 32], T());
      Fv<V> d;
      gates(dt, A, A2, d, a[r]);
      u[r] = d * (b * x);
      if (RESET && ((cut >> r) & 1)) {
        m.H = u[r];
        m.P = all<V>(-1.f);
      } else {
        m.H = fma(a[r], m.H, u[r]);
        if (!RESET || !(m.P.v[0] < 0.f)) m.P = m.P * a[r];
      }
    }
    __syncwarp();
    st_map<V>(mine, lane, m);
    __syncthreads();

    const Tile nt = s_next[s ^ 1];
    if (nt.x >= 0) stage(nt, s ^ 1);

    // the tile's map, published; then the state entering the tile
    Fv<V> h;
#pragma unroll
    for (int i = 0; i < V; ++i) h.v[i] = p.h0 && cl + i < nc ? p.h0[(int64_t)t.z * p.ds + t.w + cl + i] : 0.f;
    if (p.ticket) {
      uint64_t* ent = p.ent + (int64_t)t.y * p.nent * CW;
      const int in_span = t.x % kSpan, span = t.x / kSpan, link = span / kSpan, in_link = span % kSpan;
      Map<V> tile_map;
      if (warp == 0) {
        tile_map = ld_map<V>(buf, lane);
#pragma unroll
        for (int k = 1; k < kWarps; ++k) tile_map = then<RESET>(tile_map, ld_map<V>(buf + k * kRegion, lane));
        if (t.x + 1 < p.NT) publish<V>(ent + (int64_t)t.x * CW, lane, tile_map);
      }
      // warps 0..3 compose the whole spans of the link that the tile is in, warps 4..7 the tiles
      // of the span that it is in, four entries each
      const int from = warp % 4 * 4, n = min(4, (warp < 4 ? in_link : in_span) - from);
      if (n > 0) {
        const int at = warp < 4 ? span_at(p.NT, link * kSpan + from) : span * kSpan + from;
        st_map<V>(mine + 512, lane, take<RESET, V>(ent + (int64_t)at * CW, cl, n, lane));
      }
      if (in_span == kSpan - 1 && t.x + 1 < p.NT && warp >= 4) {
        // the end of a span: its map is published before this tile waits for earlier spans, or
        // each span would wait for the one before
        named_bar_sync(1, 128);
        if (warp == 4) {
          Map<V> sp = ld_map<V>(buf + 4 * kRegion + 512, lane);
#pragma unroll
          for (int k = 5; k < kWarps; ++k) sp = then<RESET>(sp, ld_map<V>(buf + k * kRegion + 512, lane));
#pragma unroll
          for (int k = 0; k < kWarps; ++k) sp = then<RESET>(sp, ld_map<V>(buf + k * kRegion, lane));
          publish<V>(ent + (int64_t)span_at(p.NT, span) * CW, lane, sp);
        }
      }
      if (link > 0) h = take<false, V>(ent + (int64_t)link_at(p.NT, link - 1) * CW, cl, 1, lane).H;
      __syncthreads();
      const int outer = (in_link + 3) / 4, inner = (in_span + 3) / 4;
      for (int k = 0; k < outer; ++k) h = apply<RESET>(ld_map<V>(buf + k * kRegion + 512, lane), h);
      for (int k = 4; k < 4 + inner; ++k) h = apply<RESET>(ld_map<V>(buf + k * kRegion + 512, lane), h);
      if (warp == 0 && in_span == kSpan - 1 && in_link == kSpan - 1 && t.x + 1 < p.NT)  // the end of a link
        publish<V>(ent + (int64_t)link_at(p.NT, link) * CW, lane, {all<V>(0.f), apply<RESET>(tile_map, h)});
    } else {
      __syncthreads();
    }
    if (p.states && warp == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (cl + i < nc) p.states[((int64_t)t.z * p.NT + t.x) * p.ds + t.w + cl + i] = h.v[i];
    }
    for (int k = 0; k < warp; ++k) h = apply<RESET>(ld_map<V>(buf + k * kRegion, lane), h);

    T* y = static_cast<T*>(p.y) + t.z * p.ysb + t0 * p.yst + t.w;
    if (p.out_vec && nv >= kRows && nc >= CW) {
      char* row = reinterpret_cast<char*>(y + cl);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        h = RESET && ((cut >> r) & 1) ? u[r] : fma(a[r], h, u[r]);
        *reinterpret_cast<uint32_t*>(row) = f_word(h);
        row += p.yst * (int64_t)sizeof(T);
      }
    } else {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        h = RESET && ((cut >> r) & 1) ? u[r] : fma(a[r], h, u[r]);
        if (r < nv) st_word<T>(y + r * p.yst, cl, nc, p.out_vec, h);
      }
    }
    if (p.h_last && t.x == p.NT - 1 && warp == kWarps - 1) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (cl + i < nc) p.h_last[(int64_t)t.z * p.ds + t.w + cl + i] = h.v[i];
    }
    t = nt;
  }
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

// ---------------------------------------------------------------- plans
// every row of a tensor (batch stride sb, row stride st, in elements) starts on `align` bytes
static int rows_allow(const void* p, int64_t sb, int64_t st, int es, int align) {
  return reinterpret_cast<uintptr_t>(p) % align == 0 && sb * es % align == 0 && st * es % align == 0;
}
static int64_t scan_entries(int64_t NT) {
  return NT + (NT + kSpan - 1) / kSpan + (NT + kSpan * kSpan - 1) / (kSpan * kSpan);
}
// the ticket, then the entries (channels rounded up to the wider of the two tiles)
static size_t scan_ws(int64_t B, int64_t L, int64_t ds) {
  const int64_t NT = (L + kStateRows - 1) / kStateRows;
  if (B < 1 || ds < 1 || NT < 2) return 0;
  return 16 + (size_t)(B * ((ds + 63) / 64 * 64)) * scan_entries(NT) * 8;
}
static void scan_plan(ScanParams& p, int CW, void* ws) {
  p.nch = (p.ds + CW - 1) / CW;
  p.NG = p.B * p.nch;
  p.ntiles = (int64_t)p.NG * p.NT;
  p.nent = (int)scan_entries(p.NT);
  p.ticket = p.NT > 1 ? static_cast<unsigned*>(ws) : nullptr;
  p.ent = p.NT > 1 ? reinterpret_cast<uint64_t*>(static_cast<char*>(ws) + 16) : nullptr;
}
static int scan_clear(const ScanParams& p, cudaStream_t s, const char* what) {
  if (!p.ticket) return 0;
  const cudaError_t e = cudaMemsetAsync(p.ticket, 0xff, scan_ws(p.B, p.L, p.ds), s);
  return e == cudaSuccess ? 0 : fail((int)e, "%s: %s", what, cudaGetErrorString(e));
}
template <typename T, bool RESET, int CB>
static void scan_fwd_launch(const ScanParams& p, cudaStream_t s) {
  constexpr int smem = 2 * kWarps * 3 * kRows * 128;
  auto k = gated_scan_fwd_kernel<T, RESET, CB>;
  cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  const int64_t most = (int64_t)num_sms() * kFwdCtas;
  k<<<(unsigned)(p.ntiles < most ? p.ntiles : most), kWarps * 32, smem, s>>>(p);
}
template <typename T>
static void scan_fwd_launch(const ScanParams& p, int cb, cudaStream_t s) {
  constexpr int least = sizeof(T) == 4 ? 4 : 0;  // fp32 rows always allow 4 bytes
  if (cb == 16) p.reset ? scan_fwd_launch<T, true, 16>(p, s) : scan_fwd_launch<T, false, 16>(p, s);
  else if (cb == 4) p.reset ? scan_fwd_launch<T, true, 4>(p, s) : scan_fwd_launch<T, false, 4>(p, s);
  else p.reset ? scan_fwd_launch<T, true, least>(p, s) : scan_fwd_launch<T, false, least>(p, s);
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
  const size_t need = scan_ws(B, L, ds);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(HDC_E_WORKSPACE, "gated_scan: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!aligned16(workspace)) return fail(HDC_E_ALIGN, "gated_scan: the workspace is not 16-byte aligned");
  if (B * ((ds + 31) / 32) > (int64_t(1) << 30) || B * ((ds + 31) / 32) * ((L + kStateRows - 1) / kStateRows) > (int64_t(1) << 31))
    return fail(HDC_E_SHAPE, "gated_scan: B=%lld x L=%lld x d_state=%lld is too large", (long long)B, (long long)L, (long long)ds);
  ScanParams p{};
  p.projs = projs; p.psb = proj_sb; p.pst = proj_st; p.A_log = A_log; p.a_bf16 = a_dtype == HDC_BF16;
  p.h0 = h0; p.reset = reset; p.y = y; p.ysb = y_sb; p.yst = y_st; p.h_last = h_last; p.states = states;
  p.B = (int)B; p.L = (int)L; p.ds = (int)ds; p.NT = (int)((L + kStateRows - 1) / kStateRows);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  if (L == 0) {  // nothing to scan: the state stays as it is
    if (!h_last) return HDC_OK;
    const cudaError_t e = h0 ? cudaMemcpyAsync(h_last, h0, (size_t)B * ds * 4, cudaMemcpyDeviceToDevice, s)
                             : cudaMemsetAsync(h_last, 0, (size_t)B * ds * 4, s);
    return e == cudaSuccess ? HDC_OK : fail((int)e, "gated_scan: %s", cudaGetErrorString(e));
  }
  const int es = dtype == HDC_F32 ? 4 : 2;
  scan_plan(p, 128 / es, workspace);
  p.out_vec = rows_allow(y, y_sb, y_st, es, 4);
  if (int e = scan_clear(p, s, "gated_scan")) return e;
  const int cb = rows_allow(projs, proj_sb, proj_st, es, 16) && ds * es % 16 == 0 ? 16
                 : rows_allow(projs, proj_sb, proj_st, es, 4) && ds * es % 4 == 0 ? 4 : 0;
  if (dtype == HDC_F32) scan_fwd_launch<float>(p, cb, s);
  else scan_fwd_launch<__nv_bfloat16>(p, cb, s);
  return launch_status("gated_scan_fwd_kernel");
}

extern "C" size_t hdc_gated_scan_workspace_bytes(int64_t B, int64_t L, int64_t ds) { return scan_ws(B, L, ds); }

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
