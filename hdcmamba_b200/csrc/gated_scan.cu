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
// Schedule of the scans (bound by HBM: 3 values read and 1 written per step and channel forward,
// 4 and 3 backward).  The sequence is cut into tiles of 64 steps x a few dozen channels.  A step
// is the map h -> a h + u, and maps compose: (P, H) then (P', H') is (P' P, P' H + H'), so each
// tile is scanned from a zero state, and the state entering it is added afterwards through P:
//   * a warp owns 8 steps of the tile, a lane a few neighbouring channels; its a and u stay in
//     registers between the local scan and the outputs, so every input is read once;
//   * the 8 warps' maps are composed through shared memory, and the tile's map is published in
//     the workspace;
//   * the state entering the tile is composed from at most 31 published entries: the state at
//     the end of the last whole 256 tiles, the maps of the whole 16-tile spans after it, and the
//     maps of the tiles after those.  Which entries is a matter of the tile's index alone, so
//     the result does not depend on timing.
// The gradient is the same scan from the end, of the maps c -> a (dy + c), on the same tiles;
// the states inside a tile are scanned again from the one that the forward saved at its start.
// CTAs take tiles by ticket, time-major: a tile waits only for tiles with smaller tickets,
// which running CTAs hold, so the waits end.  They are bounded all the same: a call whose wait
// runs out ends soon (a word of its workspace says so to its other waits), reports it, and what
// the missing entry would have reached is NaN; later calls know nothing of it.  An entry is one
// 64-bit word per channel, (P, H); the workspace is set to all ones before the launch, which
// no published P is, so the word is its own flag.  The next tile is in flight (cp.async)
// while one is computed.
// P < 0 marks a map that a reset has cut off from what came before (P is otherwise >= 0).
//
// Why tiles of 64 steps: what a tile keeps between its two halves (a and u: 8 bytes per step and
// channel) has to stay on the SM, in registers, and 16 to 32 warps of it fill them.  Measured
// (device time, inputs out of L2, against 6550 GB/s): 8 x 4096 x 1280 bf16 forward 94 us (54%),
// backward 175 us (51%); 1 x 32768 x 768 bf16 forward 93 us (33%); 1 x 32768 x 64 bf16 17 us;
// 3 x 1537 x 333 fp32 forward 17 us, backward 29 us.  With many channels nothing is saturated: 16
// warps of dependent instructions, with the barriers and the loads between them, fill 54 to 57% of the
// issue slots (without the exchange the forward takes 44 us per 201 MB); with few channels each
// round of tiles waits for the slowest map before it, some 4 us of a round's 8.  Tried and slower: tickets that run the maps a
// few hundred tiles ahead of the outputs (inputs read again from L2: 105 us for 91), one word per
// lane everywhere (scan_words), three backward CTAs per SM (spills).
#include <atomic>
#include <type_traits>

#include "tc.cuh"
#include "vec.cuh"

namespace hdc {

constexpr int kStateRows = 64;       // rows per tile = rows per saved state
constexpr int kWarps = 8, kRows = 8;  // warps per tile, steps per warp
constexpr int kSpan = 16;            // tiles per span, spans per chain link
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
  float* dA_part;   // [NT][NG][CW]: each tile's sum of s d
  float* dh0;
  int B, L, ds, NT;
  // tiles
  int nch;          // channel groups
  int NG;           // channel groups of all batches
  int64_t ntiles;   // NG * NT
  unsigned* ticket;  // NULL: a single tile in time, taken by block index, nothing published
                     // ticket[kGaveUp]: all ones, 0 once a wait of this call has run out
  uint64_t* ent;    // [NG][NT + spans + links][CW] published entries
  int nent;         // entries per group
  uint64_t div_NG, div_nch;  // 2^64 / d rounded up (0: d = 1)
  int CW;           // channels per tile
  int out_vec;      // the outputs' rows allow whole lanes
};

__device__ __forceinline__ float ld_param(const void* p, int bf16, int i) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

// softplus with the Block's threshold (hdcmamba/model.py:192), exact for small exp(x) too
__device__ __forceinline__ float softplus_acc(float x) { return x > 20.0f ? x : log1pf(expf(x)); }

// ---------------------------------------------------------------- a lane's channels
// V neighbouring channels of a lane: W words of 4 bytes (fp32: V = W, bf16: V = 2 W), computed
// as pairs where V is even (fma.rn.f32x2 and friends: two fp32 operations per issued instruction).
template <typename T, int W> constexpr int kV = W * 4 / (int)sizeof(T);

// a lane's channels from and to its words
template <typename T, int W> __device__ __forceinline__ Fv<kV<T, W>> ld_words(const char* p) {
  uint32_t w[W];
  if constexpr (W == 2) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    w[0] = q.x; w[1] = q.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  Fv<kV<T, W>> r;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (sizeof(T) == 4) {
      r.v[i] = __uint_as_float(w[i]);
    } else {
      r.v[2 * i] = __uint_as_float(w[i] << 16);
      r.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  return r;
}
template <typename T, int W> __device__ __forceinline__ void st_words(void* p, const Fv<kV<T, W>>& f) {
  uint32_t w[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(f.v[i]);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f.v[2 * i], f.v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  if constexpr (W == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}
// channels c, c+1, ... (those < nc) of a row; vec: the row allows whole lanes
template <typename T, int W>
__device__ __forceinline__ void st_row(T* row, int c, int nc, int vec, const Fv<kV<T, W>>& f) {
  if (vec && c + kV<T, W> <= nc) {
    st_words<T, W>(row + c, f);
  } else {
#pragma unroll
    for (int i = 0; i < kV<T, W>; ++i)
      if (c + i < nc) row[c + i] = from_f<T>(f.v[i]);
  }
}
// a word of dt = -inf
template <typename T> constexpr uint32_t kNoStep = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;

// d = softplus(x).
//   fp32: the library's exp and log1p.
//   bf16 inputs: softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) by the hardware's 2^x, and
//   log1p(e) = e p(e) on [0, 1] with p of degree 7, fitted here for the least relative error
//   (weighted least squares on Chebyshev points, weights iterated to equal errors: 2e-7, 3e-7
//   with fp32 evaluation; the bf16 input itself is 2^-9 off).  e p(e) keeps its relative accuracy
//   for small e, where log(1 + e) loses it.
template <typename T, int V> __device__ __forceinline__ Fv<V> gate(const Fv<V>& x) {
  if constexpr (sizeof(T) == 4) {
    Fv<V> d;
#pragma unroll
    for (int i = 0; i < V; ++i) d.v[i] = softplus_acc(x.v[i]);
    return d;
  } else {
    Fv<V> e, m;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      e.v[i] = ex2(-1.4426950408889634f * fabsf(x.v[i]));
      asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(m.v[i]) : "f"(x.v[i]));  // NaN stays NaN
    }
    Fv<V> p = all<V>(-0.008539206348359585f);
    p = fma(p, e, all<V>(0.04408962279558182f));
    p = fma(p, e, all<V>(-0.10768169909715652f));
    p = fma(p, e, all<V>(0.17745240032672882f));
    p = fma(p, e, all<V>(-0.24495463073253632f));
    p = fma(p, e, all<V>(0.33275479078292847f));
    p = fma(p, e, all<V>(-0.4999740421772003f));
    p = fma(p, e, all<V>(0.9999998211860657f));
    return fma(p, e, m);
  }
}
// A = -exp(A_log), kept finite: -inf times the closed gate of a step past the end (d = 0) would be
// NaN, and its decay is 1 (NaN stays NaN)
__device__ __forceinline__ float finite_rate(float A) { return A < -3.402823466e38f ? -3.402823466e38f : A; }
template <typename T> __device__ __forceinline__ float rate(float A_log) {
  return finite_rate(sizeof(T) == 4 ? -expf(A_log) : -ex2(1.4426950408889634f * A_log));
}
// a = exp(d A), by the library's exp in both types: its error compounds over the steps that a
// state remembers, and the hardware's 2^x doubles the error of the fp32 states and of dA_log (8 x
// 4096 x 1280 bf16 forward 87 us with it, 94 without; backward 168 and 174).
template <int V> __device__ __forceinline__ Fv<V> decay(const Fv<V>& d, const Fv<V>& A) {
  const Fv<V> l = d * A;
  Fv<V> a;
#pragma unroll
  for (int i = 0; i < V; ++i) a.v[i] = expf(l.v[i]);
  return a;
}
// sigmoid(x) = 1 / (1 + exp(-x)); bf16: 0 where exp(-x) overflows (x < -88)
template <typename T, int V> __device__ __forceinline__ Fv<V> sigmoid(const Fv<V>& x) {
  Fv<V> s;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] = 1.f / (1.f + expf(-x.v[i]));
  } else {
    s = x * all<V>(-1.4426950408889634f);
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] = ex2(s.v[i]);
    s = s + all<V>(1.f);
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] = rcp(s.v[i]);
  }
  return s;
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
// a lane's V values in shared memory, slot k of arrays of 32 lanes
template <int V> __device__ __forceinline__ void st_f(char* p, int k, int lane, const Fv<V>& f) {
  float* q = reinterpret_cast<float*>(p) + (k * 32 + lane) * V;
  if constexpr (V == 4) *reinterpret_cast<float4*>(q) = make_float4(f.v[0], f.v[1], f.v[2], f.v[3]);
  else if constexpr (V == 2) *reinterpret_cast<float2*>(q) = make_float2(f.v[0], f.v[1]);
  else *q = f.v[0];
}
template <int V> __device__ __forceinline__ Fv<V> ld_f(const char* p, int k, int lane) {
  const float* q = reinterpret_cast<const float*>(p) + (k * 32 + lane) * V;
  if constexpr (V == 4) {
    const float4 t = *reinterpret_cast<const float4*>(q);
    return {{t.x, t.y, t.z, t.w}};
  } else if constexpr (V == 2) {
    const float2 t = *reinterpret_cast<const float2*>(q);
    return {{t.x, t.y}};
  } else {
    return {{*q}};
  }
}
// a map in the slots k and k + 1
template <int V> constexpr int kMapBytes = 2 * 32 * V * 4;
template <int V> __device__ __forceinline__ void st_map(char* p, int lane, const Map<V>& m) {
  st_f<V>(p, 0, lane, m.P);
  st_f<V>(p, 1, lane, m.H);
}
template <int V> __device__ __forceinline__ Map<V> ld_map(const char* p, int lane) {
  return {ld_f<V>(p, 0, lane), ld_f<V>(p, 1, lane)};
}

// ---------------------------------------------------------------- published entries
constexpr uint32_t kUnset = 0xffffffffu;  // P of a word that is not published
// entry e (its first word), the lane's words
template <int V> __device__ __forceinline__ void publish(uint64_t* e, int lane, const Map<V>& m) {
  uint64_t w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    uint32_t P = __float_as_uint(m.P.v[i]);
    if (P == kUnset) P = 0x7fffffffu;  // a NaN stays one
    w[i] = ((uint64_t)__float_as_uint(m.H.v[i]) << 32) | P;
  }
  if constexpr (V == 1) {
    asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(e + lane), "l"(w[0]) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2)
      asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(e + lane * V + i), "l"(w[i]), "l"(w[i + 1])
                   : "memory");
  }
}
template <int V> __device__ __forceinline__ void ld_entry(const uint64_t* e, uint64_t (&w)[V]) {
  if constexpr (V == 1) {
    asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(w[0]) : "l"(e) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2)
      asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(w[i]), "=l"(w[i + 1]) : "l"(e + i) : "memory");
  }
}
// The limit of a wait in clock cycles, some 2 per ns (a variable of the device and not a parameter of
// the launch: read only while waiting, it leaves the rest of the kernel as it is; gradient of 8 x
// 4096 x 1280 184 us as a parameter, 180 so).
constexpr long long kMostWaitNs = 2000000000ll;
static __device__ long long g_wait_cycles = 2 * kMostWaitNs;
constexpr int kGaveUp = 1;  // word of the workspace's header
// Compose n in 1..4 neighbouring entries, waited for (up to the limit, then error 61; what is
// missing then is NaN).  e: entry 0 of them.  While an entry is missing, one word of each is
// polled, not the whole entries.
template <bool RESET, int V>
__device__ __forceinline__ Map<V> take(const ScanParams& p, const uint64_t* e, int n, int lane) {
  uint64_t w[4][V];
  long long t0 = 0;
  while (true) {
    bool ok = true;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) ld_entry<V>(e + (k * 32 + lane) * V, w[k]);
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
        ld_entry<1>(e + lane * 32 * V, one);
        // a wait of this call that has run out elsewhere ends this one too (looked at after some
        // 0.1 ms only: waits are of a few us, and the word lies beside the ticket)
        const long long waited = clock64() - t0;
        late = waited >= *static_cast<volatile long long*>(&g_wait_cycles) ||
               (waited > 200000 && *static_cast<volatile unsigned*>(p.ticket + kGaveUp) == 0);
      } while ((uint32_t)one[0] == kUnset && !late);
    }
    if (__any_sync(0xffffffffu, late)) {
      if (lane == 0) {
        atomicExch(p.ticket + kGaveUp, 0u);
        atomicCAS(&g_dev_error, 0, 61);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if ((uint32_t)w[k][i] == kUnset) w[k][i] = 0x7fffffff7fffffffull;
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

// The composition of the 8 warps' maps, and its publication by one warp.
template <bool RESET, bool REV, int V> __device__ __forceinline__ Map<V> tile_map_of(const char* maps, int stride, int lane) {
  Map<V> m = ld_map<V>(maps + (REV ? kWarps - 1 : 0) * stride, lane);
#pragma unroll
  for (int k = 1; k < kWarps; ++k) m = then<RESET>(m, ld_map<V>(maps + (REV ? kWarps - 1 - k : k) * stride, lane));
  return m;
}
template <bool RESET, bool REV, int V>
__device__ __forceinline__ void publish_tile(const ScanParams& p, int g, int q, const char* maps, int stride, int lane) {
  if (q + 1 < p.NT)
    publish<V>(p.ent + ((int64_t)g * p.nent + q) * 32 * V, lane, tile_map_of<RESET, REV, V>(maps, stride, lane));
}

// The exchange between tiles, the same for both directions.  q: the tile's index in the order
// of the scan.  maps: the 8 warps' maps in shared memory, warp w's at maps + w * stride, composed
// in the order of the scan (REV: from the last warp to the first).  pre: this warp's slot at
// pre + warp * pre_stride.  All threads call it (it synchronises the CTA once, after the maps'
// own barrier); h: the state entering the sequence, returned as the state entering the tile.
template <bool RESET, bool REV, int V>
__device__ __forceinline__ Fv<V> enter_tile(const ScanParams& p, int g, int q, const char* maps, int stride, char* pre,
                                            int pre_stride, Fv<V> h, int warp, int lane) {
  constexpr int CW = 32 * V;
  uint64_t* ent = p.ent + (int64_t)g * p.nent * CW;
  // entries of a group: tiles, then spans of 16 tiles, then links of 16 spans (P unused, H the
  // state at their end)
  uint64_t* spans = ent + (int64_t)p.NT * CW;
  uint64_t* links = spans + (int64_t)((p.NT + kSpan - 1) / kSpan) * CW;
  const int in_span = q % kSpan, span = q / kSpan, link = span / kSpan, in_link = span % kSpan;
  const bool more = q + 1 < p.NT;
  auto tile_map = [&]() { return tile_map_of<RESET, REV, V>(maps, stride, lane); };
  // warps 0..3 compose the whole spans of the link that the tile is in, warps 4..7 the tiles of
  // the span that it is in, four entries each
  const int from = warp % 4 * 4, n = min(4, (warp < 4 ? in_link : in_span) - from);
  if (n > 0) {
    const uint64_t* e = warp < 4 ? spans + (int64_t)(link * kSpan + from) * CW : ent + (int64_t)(span * kSpan + from) * CW;
    st_map<V>(pre + warp * pre_stride, lane, take<RESET, V>(p, e, n, lane));
  }
  if (in_span == kSpan - 1 && more && warp >= 4) {
    // the end of a span: its map is published before this tile waits for earlier spans, or
    // each span would wait for the one before
    named_bar_sync(1, 128);
    if (warp == 4) {
      Map<V> m = ld_map<V>(pre + 4 * pre_stride, lane);
#pragma unroll
      for (int k = 5; k < kWarps; ++k) m = then<RESET>(m, ld_map<V>(pre + k * pre_stride, lane));
      publish<V>(spans + (int64_t)span * CW, lane, then<RESET>(m, tile_map()));
    }
  }
  if (link > 0) h = take<false, V>(p, links + (int64_t)(link - 1) * CW, 1, lane).H;
  __syncthreads();
  const int outer = (in_link + 3) / 4, inner = (in_span + 3) / 4;
  for (int k = 0; k < outer; ++k) h = apply<RESET>(ld_map<V>(pre + k * pre_stride, lane), h);
  for (int k = 4; k < 4 + inner; ++k) h = apply<RESET>(ld_map<V>(pre + k * pre_stride, lane), h);
  if (warp == 0 && in_span == kSpan - 1 && in_link == kSpan - 1 && more)  // the end of a link
    publish<V>(links + (int64_t)link * CW, lane, {all<V>(0.f), apply<RESET>(tile_map(), h)});
  return h;
}

// ---------------------------------------------------------------- staging
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool ok, std::integral_constant<int, 16>) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool ok, std::integral_constant<int, 4>) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Copies of one warp's 8 rows (128 W bytes each) of a tile, rows >= nv and channels >= nc as
// zeros.  CB: bytes per copy (16 or 4, as the rows allow), or 0: element by element, not
// asynchronous.
template <typename T, int W, int CB> struct Rows {
  static constexpr int kBytes = 128 * W, kCopy = CB ? CB : 4;
  static constexpr int kPer = kBytes / kCopy;               // copies per row
  static constexpr int kAt = kPer < 32 ? 32 / kPer : 1;     // rows per warp-wide copy
  static constexpr int kX = kPer > 32 ? kPer / 32 : 1;      // warp-wide copies per row
  int r0, x;  // the lane's first row and first byte of a row
  __device__ explicit Rows(int lane) : r0(kPer < 32 ? lane / kPer : 0), x((kPer < 32 ? lane % kPer : lane) * kCopy) {}
  // tile: the tile's first element; row0: the warp's first row in it; st: row stride (elements);
  // `arrays` consecutive regions, their sources `apart` elements from each other
  template <int arrays>
  __device__ __forceinline__ void copy(char* region, const T* tile, int row0, int64_t st, int64_t apart, int nv,
                                       int nc) const {
#pragma unroll
    for (int i = 0; i < kRows / kAt; ++i)
#pragma unroll
      for (int j = 0; j < kX; ++j) {
        const int r = r0 + i * kAt, xb = x + j * 32 * kCopy;
        const bool ok = r < nv && xb < nc * (int)sizeof(T);
        if constexpr (CB == 0) {
          constexpr int per = 4 / (int)sizeof(T);
          const int c = xb / (int)sizeof(T);
#pragma unroll
          for (int k = 0; k < arrays; ++k)
#pragma unroll
            for (int e = 0; e < per; ++e)
              reinterpret_cast<T*>(region + (k * kRows + r) * kBytes)[c + e] =
                  r < nv && c + e < nc ? tile[k * apart + (row0 + r) * st + c + e] : from_f<T>(0.f);
        } else {
          const char* src = reinterpret_cast<const char*>(tile) + (ok ? (row0 + r) * st * (int64_t)sizeof(T) + xb : 0);
          const uint32_t dst = smem_u32(region) + r * kBytes + xb;
#pragma unroll
          for (int k = 0; k < arrays; ++k)
            cp_async(dst + k * kRows * kBytes, src + k * apart * (int64_t)sizeof(T), ok, std::integral_constant<int, CB>());
        }
      }
  }
};

// n / d for n, d < 2^32 from m = 2^64 / d rounded up: n m = 2^64 n/d + n e with e < d, n e < 2^64
__device__ __forceinline__ unsigned quotient(unsigned n, uint64_t m) { return m ? (unsigned)__umul64hi(m, n) : n; }

// A tile as broadcast through shared memory: index in the scan's order, group, batch, first
// channel; x < 0: none
using Tile = int4;
__device__ __forceinline__ Tile tile_of(const ScanParams& p, int64_t id, int CW) {
  if (id >= p.ntiles) return make_int4(-1, 0, 0, 0);
  const unsigned q = quotient((unsigned)id, p.div_NG), g = (unsigned)id - q * p.NG, b = quotient(g, p.div_nch);
  return make_int4((int)q, (int)g, (int)b, (int)(g - b * p.nch) * CW);
}
__device__ __forceinline__ int64_t next_tile(const ScanParams& p, int64_t last) {
  if (!p.ticket) return last + gridDim.x;
  return (int64_t)(unsigned)(atomicAdd(p.ticket, 1u) + 1u);  // the counter starts at all ones
}
// the lane's channels of a [.., ds] fp32 row (nc of them in the tile), zeros where there is none
template <int V> __device__ __forceinline__ Fv<V> ld_state(const float* row, int cl, int nc) {
  Fv<V> h;
#pragma unroll
  for (int i = 0; i < V; ++i) h.v[i] = row && cl + i < nc ? row[cl + i] : 0.f;
  return h;
}
template <int V> __device__ __forceinline__ void st_state(float* row, int cl, int nc, const Fv<V>& h) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (cl + i < nc) row[cl + i] = h.v[i];
}

// Resident forward CTAs per SM.  Two words per lane need 128 registers; one needs 64 in bf16 (32768 x
// 64: 15.1 us with four, 16.7 with three) and more in fp32 (3 x 1537 x 333: 17.0 us with three, 19.3
// with four).
template <typename T, int W> constexpr int kFwdCtas = W == 2 ? 2 : sizeof(T) == 4 ? 3 : 4;

template <typename T, int W, bool RESET, int CB>
__global__ void __launch_bounds__(kWarps * 32, kFwdCtas<T, W>) gated_scan_fwd_kernel(const __grid_constant__ ScanParams p) {
  constexpr int V = kV<T, W>, CW = 32 * V, RB = 128 * W, kRegion = 3 * kRows * RB;
  static_assert(2 * kMapBytes<V> <= kRegion, "maps fit into a warp's staged rows");
  extern __shared__ __align__(128) char raw[];  // [2][warp][dt, x, b][row][RB bytes]
  __shared__ Tile s_next[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cl = lane * V;  // the lane's first channel of the tile
  const Rows<T, W, CB> rows(lane);
  int64_t id = 0;  // thread 0's

  // of the staged tile: the reset flag of step `lane` of the warp, A_log of the lane's channels
  uint32_t rb = 0;
  Fv<V> A_next = all<V>(0.f);
  auto stage = [&](const Tile& t, int s) {
    const int t0 = t.x * kStateRows, nv = p.L - t0 - warp * kRows, nc = p.ds - t.w;
    const T* tile = static_cast<const T*>(p.projs) + t.z * p.psb + t0 * p.pst + t.w;
    rows.template copy<3>(raw + (s * kWarps + warp) * kRegion, tile, warp * kRows, p.pst, p.ds, nv, nc);
    cp_commit();
    if (RESET) rb = lane < min(nv, kRows) ? p.reset[(int64_t)t.z * p.L + t0 + warp * kRows + lane] : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) A_next.v[i] = cl + i < nc ? ld_param(p.A_log, p.a_bf16, t.w + cl + i) : 0.f;
  };

  if (threadIdx.x == 0) {
    id = p.ticket ? next_tile(p, 0) : blockIdx.x;
    s_next[0] = tile_of(p, id, CW);
  }
  __syncthreads();
  Tile t = s_next[0];
  if (t.x >= 0) stage(t, 0);
  bool first = true;
  for (int s = 0; t.x >= 0; s ^= 1) {
    // The tile after this one is known by now (its ticket was taken during the tile before), except
    // the first time, and then it is asked for only after the loads: a CTA that starts early
    // would else take two neighbouring tiles, and the tiles after the second one would wait until
    // it is done with the first.
    if (first) {
      cp_wait_all();
      if (threadIdx.x == 0) {
        id = next_tile(p, id);
        s_next[1] = tile_of(p, id, CW);
      }
      first = false;
    }
    char* buf = raw + s * kWarps * kRegion;
    char* mine = buf + warp * kRegion;
    const int t0 = t.x * kStateRows + warp * kRows, nv = p.L - t0, nc = p.ds - t.w;
    const uint32_t cut = RESET ? __ballot_sync(0xffffffffu, rb != 0) : 0;
    Fv<V> A;
#pragma unroll
    for (int i = 0; i < V; ++i) A.v[i] = rate<T>(A_next.v[i]);
    cp_wait_all();
    __syncwarp();
    if (nv < kRows) {  // steps past the end: dt = -inf (and x = b = 0) is the identity, a = 1, u = 0
      for (int r = max(nv, 0); r < kRows; ++r)
#pragma unroll
        for (int k = 0; k < W; ++k) reinterpret_cast<uint32_t*>(mine + r * RB)[lane * W + k] = kNoStep<T>;
    }

    // local scan of the warp's steps from a zero state
    Fv<V> a[kRows], u[kRows];
    Map<V> m = identity_map<V>();
    const char* w = mine + lane * 4 * W;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const Fv<V> dt = ld_words<T, W>(w + r * RB), x = ld_words<T, W>(w + (kRows + r) * RB);
      const Fv<V> b = ld_words<T, W>(w + (2 * kRows + r) * RB);
      const Fv<V> d = gate<T>(dt);
      a[r] = decay(d, A);
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
    if (threadIdx.x == 0) id = next_tile(p, id);
    if (p.ticket && warp == 0) publish_tile<RESET, false, V>(p, t.y, t.x, buf, kRegion, lane);
    if (nt.x >= 0) stage(nt, s ^ 1);

    // the state entering the tile, then the warp's steps
    const int64_t at = (int64_t)t.z * p.ds + t.w;
    Fv<V> h = ld_state<V>(p.h0 ? p.h0 + at : nullptr, cl, nc);
    if (p.ticket)
      h = enter_tile<RESET, false, V>(p, t.y, t.x, buf, kRegion, buf + kMapBytes<V>, kRegion, h, warp, lane);
    if (p.states && warp == 0) st_state<V>(p.states + ((int64_t)t.z * p.NT + t.x) * p.ds + t.w, cl, nc, h);
    for (int k = 0; k < warp; ++k) h = apply<RESET>(ld_map<V>(buf + k * kRegion, lane), h);

    T* y = static_cast<T*>(p.y) + t.z * p.ysb + t0 * p.yst + t.w;
    if (p.out_vec && nv >= kRows && nc >= CW) {
      char* row = reinterpret_cast<char*>(y + cl);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        h = RESET && ((cut >> r) & 1) ? u[r] : fma(a[r], h, u[r]);
        st_words<T, W>(row, h);
        row += p.yst * (int64_t)sizeof(T);
      }
    } else {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        h = RESET && ((cut >> r) & 1) ? u[r] : fma(a[r], h, u[r]);
        if (r < nv) st_row<T, W>(y + r * p.yst, cl, nc, p.out_vec, h);
      }
    }
    if (p.h_last && t.x == p.NT - 1 && warp == kWarps - 1) st_state<V>(p.h_last + at, cl, nc, h);
    if (threadIdx.x == 0) s_next[s] = tile_of(p, id, CW);
    t = nt;
  }
}

// resident backward CTAs per SM (three: 80 registers and spills, 244 us for 184, 8 x 4096 x 1280)
constexpr int kBwdCtas = 2;
// shared memory of the backward: two staged tiles, the warps' forward maps and backward maps
// (P shared), the exchange's slots, the warps' sums for dA
template <int V, int W> constexpr int kBwdMaps = 2 * kWarps * 4 * kRows * 128 * W;
template <int V, int W> constexpr int kBwdSmem = kBwdMaps<V, W> + kWarps * 32 * V * (16 + 8 + 4);

template <typename T, int W, bool RESET, int CB>
__global__ void __launch_bounds__(kWarps * 32, kBwdCtas) gated_scan_bwd_kernel(const __grid_constant__ ScanParams p) {
  constexpr int V = kV<T, W>, CW = 32 * V, RB = 128 * W, kRegion = 4 * kRows * RB;
  extern __shared__ __align__(128) char raw[];  // [2][warp][dt, x, b, dy][row][RB bytes]
  char* fmap = raw + kBwdMaps<V, W>;            // [warp] forward maps (P, H)
  char* bmap = fmap + kWarps * kMapBytes<V>;    // [warp] backward maps (P, C)
  char* pre = bmap + kWarps * kMapBytes<V>;     // [warp] exchange
  char* sums = pre + kWarps * kMapBytes<V>;     // [warp] sums of s d
  __shared__ Tile s_next[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cl = lane * V;
  const Rows<T, W, CB> rows(lane);
  int64_t id = 0;  // thread 0's

  uint32_t rb = 0;
  Fv<V> A_next = all<V>(0.f);
  auto stage = [&](const Tile& t, int s) {
    const int t0 = (p.NT - 1 - t.x) * kStateRows, nv = p.L - t0 - warp * kRows, nc = p.ds - t.w;
    char* reg = raw + (s * kWarps + warp) * kRegion;
    const T* tile = static_cast<const T*>(p.projs) + t.z * p.psb + t0 * p.pst + t.w;
    rows.template copy<3>(reg, tile, warp * kRows, p.pst, p.ds, nv, nc);
    const T* dyt = static_cast<const T*>(p.dy) + t.z * p.dsb + t0 * p.dst + t.w;
    rows.template copy<1>(reg + 3 * kRows * RB, dyt, warp * kRows, p.dst, 0, nv, nc);
    cp_commit();
    if (RESET) rb = lane < min(nv, kRows) ? p.reset[(int64_t)t.z * p.L + t0 + warp * kRows + lane] : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) A_next.v[i] = cl + i < nc ? ld_param(p.A_log, p.a_bf16, t.w + cl + i) : 0.f;
  };
  // the sum of the warps' s d of the tile before, in their order
  auto write_dA = [&](const Tile& t) {
    Fv<V> v = ld_f<V>(sums, 0, lane);
#pragma unroll
    for (int k = 1; k < kWarps; ++k) v = v + ld_f<V>(sums, k, lane);
    st_f<V>(reinterpret_cast<char*>(p.dA_part + ((int64_t)t.x * p.NG + t.y) * CW), 0, lane, v);
  };

  if (threadIdx.x == 0) {
    id = p.ticket ? next_tile(p, 0) : blockIdx.x;
    s_next[0] = tile_of(p, id, CW);
  }
  __syncthreads();
  Tile t = s_next[0], before = make_int4(-1, 0, 0, 0);
  if (t.x >= 0) stage(t, 0);
  for (int s = 0; t.x >= 0; s ^= 1) {
    if (before.x < 0) {  // the first time, as in the forward
      cp_wait_all();
      if (threadIdx.x == 0) {
        id = next_tile(p, id);
        s_next[1] = tile_of(p, id, CW);
      }
    }
    char* mine = raw + (s * kWarps + warp) * kRegion;
    const int tt = p.NT - 1 - t.x, t0 = tt * kStateRows + warp * kRows, nv = p.L - t0, nc = p.ds - t.w;
    const uint32_t cut = RESET ? __ballot_sync(0xffffffffu, rb != 0) : 0;
    Fv<V> h = ld_state<V>(p.states + ((int64_t)t.z * p.NT + tt) * p.ds + t.w, cl, nc);
    Fv<V> A;
#pragma unroll
    for (int i = 0; i < V; ++i) A.v[i] = rate<T>(A_next.v[i]);
    cp_wait_all();
    __syncwarp();
    if (nv < kRows) {  // steps past the end are the identity
      for (int r = max(nv, 0); r < kRows; ++r)
#pragma unroll
        for (int k = 0; k < W; ++k) reinterpret_cast<uint32_t*>(mine + r * RB)[lane * W + k] = kNoStep<T>;
    }

    // local scans of the warp's steps, forward and backward
    Fv<V> a[kRows], d[kRows], bx[kRows];
    Map<V> m = identity_map<V>();
    Fv<V> c = all<V>(0.f);
    const char* w = mine + lane * 4 * W;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const Fv<V> dt = ld_words<T, W>(w + r * RB), x = ld_words<T, W>(w + (kRows + r) * RB);
      const Fv<V> b = ld_words<T, W>(w + (2 * kRows + r) * RB);
      d[r] = gate<T>(dt);
      a[r] = decay(d[r], A);
      bx[r] = b * x;
      const Fv<V> u = d[r] * bx[r];
      // the backward map from zero: c = sum of dy_r times the decays up to step r, until a reset
      if (RESET && ((cut >> r) & 1)) {
        m.H = u;
        m.P = all<V>(-1.f);
      } else {
        m.H = fma(a[r], m.H, u);
        if (!RESET || !(m.P.v[0] < 0.f)) {
          m.P = m.P * a[r];
          c = fma(m.P, ld_words<T, W>(w + (3 * kRows + r) * RB), c);
        }
      }
    }
    st_map<V>(fmap + warp * kMapBytes<V>, lane, m);
    st_map<V>(bmap + warp * kMapBytes<V>, lane, {m.P, c});
    __syncthreads();

    const Tile nt = s_next[s ^ 1];
    if (threadIdx.x == 0) id = next_tile(p, id);
    if (p.ticket && warp == 0) publish_tile<RESET, true, V>(p, t.y, t.x, bmap, kMapBytes<V>, lane);
    if (nt.x >= 0) stage(nt, s ^ 1);
    if (warp == 2 && before.x >= 0) write_dA(before);

    // what enters the tile from its end, then the warp's part of both scans
    const int64_t at = (int64_t)t.z * p.ds + t.w;
    c = ld_state<V>(p.dh_last ? p.dh_last + at : nullptr, cl, nc);
    for (int k = 0; k < warp; ++k) h = apply<RESET>(ld_map<V>(fmap + k * kMapBytes<V>, lane), h);
    if (p.ticket) c = enter_tile<RESET, true, V>(p, t.y, t.x, bmap, kMapBytes<V>, pre, kMapBytes<V>, c, warp, lane);
    else __syncthreads();  // the sums of the tile before
    for (int k = kWarps - 1; k > warp; --k) c = apply<RESET>(ld_map<V>(bmap + k * kMapBytes<V>, lane), c);

    Fv<V> q[kRows];  // a_t h_{t-1}, 0 at a reset
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      q[r] = RESET && ((cut >> r) & 1) ? all<V>(0.f) : a[r] * h;
      h = fma(d[r], bx[r], q[r]);
    }
    Fv<V> sum = all<V>(0.f);
    T* out = static_cast<T*>(p.dprojs) + t.z * p.gsb + t0 * p.gst + t.w;
    const bool whole = p.out_vec && nv >= kRows && nc >= CW;
#pragma unroll
    for (int r = kRows - 1; r >= 0; --r) {
      const Fv<V> dt = ld_words<T, W>(w + r * RB), x = ld_words<T, W>(w + (kRows + r) * RB);
      const Fv<V> b = ld_words<T, W>(w + (2 * kRows + r) * RB);
      const Fv<V> g = ld_words<T, W>(w + (3 * kRows + r) * RB) + c;
      c = a[r] * g;
      if (RESET && ((cut >> r) & 1)) c = all<V>(0.f);
      const Fv<V> gd = g * d[r], sr = g * q[r];
      const Fv<V> ddt = fma(sr, A, g * bx[r]) * sigmoid<T>(dt);
      if (whole) {
        sum = fma(sr, d[r], sum);
        T* o = out + r * p.gst + cl;
        st_words<T, W>(o, ddt);
        st_words<T, W>(o + p.ds, gd * b);
        st_words<T, W>(o + 2 * p.ds, gd * x);
      } else if (r < nv) {
        sum = fma(sr, d[r], sum);
        T* o = out + r * p.gst;
        st_row<T, W>(o, cl, nc, p.out_vec, ddt);
        st_row<T, W>(o + p.ds, cl, nc, p.out_vec, gd * b);
        st_row<T, W>(o + 2 * p.ds, cl, nc, p.out_vec, gd * x);
      }
    }
    if (p.dh0 && tt == 0 && warp == 0) st_state<V>(p.dh0 + at, cl, nc, c);
    st_f<V>(sums, warp, lane, sum);
    if (threadIdx.x == 0) s_next[s] = tile_of(p, id, CW);
    __syncthreads();  // the maps and slots are read, the sums written
    before = t;
    t = nt;
  }
  if (warp == 2 && before.x >= 0) write_dA(before);
}

// dA_log[j] = A_j times the sum of the parts ([q][b][channel], channels padded to cpad), in their
// order: 32 strands per channel (32 channels a CTA), then the strands.
__global__ void __launch_bounds__(1024) gated_scan_dA_kernel(const float* part, int64_t parts, int cpad, int ds,
                                                             const void* A_log, int a_bf16, void* dA) {
  __shared__ float s[32][33];
  const int x = threadIdx.x & 31, k = threadIdx.x >> 5, j = blockIdx.x * 32 + x;
  float v = 0.f;
  if (j < ds) {
#pragma unroll 8
    for (int64_t i = k; i < parts; i += 32) v += part[i * cpad + j];
  }
  s[k][x] = v;
  __syncthreads();
  if (k != 0 || j >= ds) return;
  for (int i = 1; i < 32; ++i) v += s[i][x];
  v *= finite_rate(-expf(ld_param(A_log, a_bf16, j)));
  if (a_bf16) static_cast<__nv_bfloat16*>(dA)[j] = __float2bfloat16_rn(v);
  else static_cast<float*>(dA)[j] = v;
}

// One step per sequence: a thread per channel, 20 bytes (bf16) each.  Bound by the launch up to a
// few hundred thousand channels (1 x 768: 1.6 us, 256 x 2048: 4.3 us, 1.3 us of it traffic).
template <typename T>
__global__ void __launch_bounds__(128) gated_step_kernel(const T* projs, int64_t psb, const void* A_log, int a_bf16,
                                                         const float* h, const uint8_t* reset, float* h_out, T* y,
                                                         int64_t ysb, int ds) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y;
  if (j >= ds) return;
  const T* r = projs + b * psb + j;
  const float A = finite_rate(-expf(ld_param(A_log, a_bf16, j)));
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
static bool rows_allow(const void* p, int64_t sb, int64_t st, int es, int align) {
  return reinterpret_cast<uintptr_t>(p) % align == 0 && sb * es % align == 0 && st * es % align == 0;
}
static int64_t tiles_in_time(int64_t L) { return (L + kStateRows - 1) / kStateRows; }
static int64_t scan_entries(int64_t NT) {
  return NT + (NT + kSpan - 1) / kSpan + (NT + kSpan * kSpan - 1) / (kSpan * kSpan);
}
// channels rounded up to the widest tile
static int64_t scan_pad(int64_t ds) { return (ds + 127) / 128 * 128; }
// the ticket and the word beside it, then the entries, each (256 bytes or more) on whole lines
constexpr int kScanHeader = 256;
static size_t scan_ws(int64_t B, int64_t L, int64_t ds) {
  const int64_t NT = tiles_in_time(L);
  if (B < 1 || ds < 1 || NT < 2) return 0;
  return kScanHeader + (size_t)(B * scan_pad(ds)) * scan_entries(NT) * 8;
}
static void scan_plan(ScanParams& p, int CW, void* ws) {
  p.CW = CW;
  p.nch = (p.ds + CW - 1) / CW;
  p.NG = p.B * p.nch;
  p.ntiles = (int64_t)p.NG * p.NT;
  p.nent = (int)scan_entries(p.NT);
  p.div_NG = p.NG > 1 ? ~uint64_t(0) / p.NG + 1 : 0;
  p.div_nch = p.nch > 1 ? ~uint64_t(0) / p.nch + 1 : 0;
  p.ticket = p.NT > 1 ? static_cast<unsigned*>(ws) : nullptr;
  p.ent = p.NT > 1 ? reinterpret_cast<uint64_t*>(static_cast<char*>(ws) + kScanHeader) : nullptr;
}
static int scan_clear(const ScanParams& p, cudaStream_t s, const char* what) {
  if (!p.ticket) return 0;
  const size_t n = kScanHeader + (size_t)p.NG * p.CW * p.nent * 8;
  const cudaError_t e = cudaMemsetAsync(p.ticket, 0xff, n, s);
  return e == cudaSuccess ? 0 : fail((int)e, "%s: %s", what, cudaGetErrorString(e));
}
// sizes that the kernels' 32-bit indices hold
static int scan_fits(const char* what, int64_t B, int64_t L, int64_t ds) {
  const int64_t groups = B * ((ds + 31) / 32);
  if (groups > (int64_t(1) << 30) || groups * tiles_in_time(L) > (int64_t(1) << 31) - 4096)
    return fail(HDC_E_SHAPE, "%s: B=%lld x L=%lld x d_state=%lld is too large", what, (long long)B, (long long)L,
                (long long)ds);
  return 0;
}
// Words per lane in the forward: in bf16 two (tiles of 128 channels) halve what a tile costs beside
// its arithmetic (us with two and with one: 8 x 4096 x 1280 94 and 101, 32 x 1024 x 512 40 and 43, 1 x
// 32768 x 768 93 and 95, 1 x 8192 x 2048 55 and 55); one where much of a wide tile would be empty (1 x
// 32768 x 64 23 and 17, 4 x 4096 x 192 20 and 17, x 320 24 and 21, x 448 30 and 26; past 512 channels
// from 4 x 4096 x 520 36 and 32 to x 601 53 and 54), and in fp32, whose exp and log1p take the registers
// (3 x 1537 x 333: 17 us with one, 19 with two).  The backward holds more per channel (two words spill 500 bytes) and
// takes one.
static int scan_words(int64_t ds, int es) { return es == 2 && (ds % 128 == 0 || ds > 512) ? 2 : 1; }

template <typename T, int W, bool RESET, int CB, bool BWD>
static void scan_launch(const ScanParams& p, cudaStream_t s) {
  constexpr int V = kV<T, W>;
  constexpr int smem = BWD ? kBwdSmem<V, W> : 2 * kWarps * 3 * kRows * 128 * W;
  const int64_t most = (int64_t)num_sms() * (BWD ? kBwdCtas : kFwdCtas<T, W>);
  const unsigned grid = (unsigned)(p.ntiles < most ? p.ntiles : most);
  auto k = [] {
    if constexpr (BWD) return gated_scan_bwd_kernel<T, W, RESET, CB>;
    else return gated_scan_fwd_kernel<T, W, RESET, CB>;
  }();
  static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is set
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  k<<<grid, kWarps * 32, smem, s>>>(p);
}
template <typename T, int W, bool BWD>
static void scan_launch(const ScanParams& p, int cb, cudaStream_t s) {
  constexpr int least = sizeof(T) == 4 ? 4 : 0;  // fp32 rows always allow 4 bytes
  if (cb == 16) p.reset ? scan_launch<T, W, true, 16, BWD>(p, s) : scan_launch<T, W, false, 16, BWD>(p, s);
  else if (cb == 4) p.reset ? scan_launch<T, W, true, 4, BWD>(p, s) : scan_launch<T, W, false, 4, BWD>(p, s);
  else p.reset ? scan_launch<T, W, true, least, BWD>(p, s) : scan_launch<T, W, false, least, BWD>(p, s);
}
template <bool BWD>
static void scan_launch(const ScanParams& p, int dtype, int W, int cb, cudaStream_t s) {
  constexpr int most = BWD ? 1 : 2;
  if (dtype == HDC_F32) scan_launch<float, 1, BWD>(p, cb, s);
  else W == 2 ? scan_launch<__nv_bfloat16, most, BWD>(p, cb, s) : scan_launch<__nv_bfloat16, 1, BWD>(p, cb, s);
}

}  // namespace hdc

using namespace hdc;

extern "C" int64_t hdc_gated_scan_state_rows(void) { return kStateRows; }

extern "C" int hdc_gated_scan_wait_limit(uint64_t ns) {
  if (ns > (uint64_t)kMostWaitNs)
    return fail(HDC_E_SHAPE, "gated_scan_wait_limit: %llu ns (at most %lld)", (unsigned long long)ns, kMostWaitNs);
  const long long cycles = 2 * (long long)ns;
  const cudaError_t e = cudaMemcpyToSymbol(g_wait_cycles, &cycles, sizeof cycles);
  return e == cudaSuccess ? HDC_OK : fail((int)e, "gated_scan_wait_limit: %s", cudaGetErrorString(e));
}

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
  if (L > 0 && !rows_apart(B, y_sb, L, y_st, ds))
    return fail(HDC_E_SHAPE, "gated_scan: y rows overlap (y_sb=%lld, y_st=%lld)", (long long)y_sb, (long long)y_st);
  const size_t need = scan_ws(B, L, ds);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(HDC_E_WORKSPACE, "gated_scan: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!aligned16(workspace)) return fail(HDC_E_ALIGN, "gated_scan: the workspace is not 16-byte aligned");
  if (int e = scan_fits("gated_scan", B, L, ds)) return e;
  ScanParams p{};
  p.projs = projs; p.psb = proj_sb; p.pst = proj_st; p.A_log = A_log; p.a_bf16 = a_dtype == HDC_BF16;
  p.h0 = h0; p.reset = reset; p.y = y; p.ysb = y_sb; p.yst = y_st; p.h_last = h_last; p.states = states;
  p.B = (int)B; p.L = (int)L; p.ds = (int)ds; p.NT = (int)tiles_in_time(L);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  if (L == 0) {  // nothing to scan: the state stays as it is
    if (!h_last) return HDC_OK;
    const cudaError_t e = h0 ? cudaMemcpyAsync(h_last, h0, (size_t)B * ds * 4, cudaMemcpyDeviceToDevice, s)
                             : cudaMemsetAsync(h_last, 0, (size_t)B * ds * 4, s);
    return e == cudaSuccess ? HDC_OK : fail((int)e, "gated_scan: %s", cudaGetErrorString(e));
  }
  const int es = dtype == HDC_F32 ? 4 : 2, W = scan_words(ds, es);
  scan_plan(p, 128 * W / es, workspace);
  p.out_vec = rows_allow(y, y_sb, y_st, es, 4 * W);
  if (int e = scan_clear(p, s, "gated_scan")) return e;
  const int cb = rows_allow(projs, proj_sb, proj_st, es, 16) && ds * es % 16 == 0 ? 16
                 : rows_allow(projs, proj_sb, proj_st, es, 4) && ds * es % 4 == 0 ? 4 : 0;
  scan_launch<false>(p, dtype, W, cb, s);
  return launch_status("gated_scan_fwd_kernel");
}

extern "C" size_t hdc_gated_scan_workspace_bytes(int64_t B, int64_t L, int64_t ds) { return scan_ws(B, L, ds); }

// the forward's, then the tiles' parts of dA
extern "C" size_t hdc_gated_scan_bwd_workspace_bytes(int64_t B, int64_t L, int64_t ds) {
  if (B < 1 || L < 1 || ds < 1) return 0;
  return scan_ws(B, L, ds) + (size_t)tiles_in_time(L) * B * scan_pad(ds) * 4;
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
  if (B > 0 && L > 0 && !rows_apart(B, dp_sb, L, dp_st, 3 * ds))
    return fail(HDC_E_SHAPE, "gated_scan_bwd: dprojs rows overlap (dp_sb=%lld, dp_st=%lld)", (long long)dp_sb,
                (long long)dp_st);
  const size_t need = hdc_gated_scan_bwd_workspace_bytes(B, L, ds);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(HDC_E_WORKSPACE, "gated_scan_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!aligned16(workspace)) return fail(HDC_E_ALIGN, "gated_scan_bwd: the workspace is not 16-byte aligned");
  if (int e = scan_fits("gated_scan_bwd", B, L, ds)) return e;
  ScanParams p{};
  p.projs = projs; p.psb = proj_sb; p.pst = proj_st; p.A_log = A_log; p.a_bf16 = a_dtype == HDC_BF16;
  p.reset = reset; p.states = const_cast<float*>(states); p.dy = dy; p.dsb = dy_sb; p.dst = dy_st;
  p.dh_last = dh_last; p.dprojs = dprojs; p.gsb = dp_sb; p.gst = dp_st; p.dh0 = dh0;
  p.B = (int)B; p.L = (int)L; p.ds = (int)ds; p.NT = (int)tiles_in_time(L);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  const int es = dtype == HDC_F32 ? 4 : 2, W = 1;
  scan_plan(p, 128 * W / es, workspace);
  if (B > 0 && L > 0) {
    p.dA_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + scan_ws(B, L, ds));
    p.out_vec = rows_allow(dprojs, dp_sb, dp_st, es, 4 * W) && ds * es % (4 * W) == 0;
    if (int e = scan_clear(p, s, "gated_scan_bwd")) return e;
    const bool in = ds * es % 4 == 0 && rows_allow(projs, proj_sb, proj_st, es, 4) && rows_allow(dy, dy_sb, dy_st, es, 4);
    const int cb = in && ds * es % 16 == 0 && rows_allow(projs, proj_sb, proj_st, es, 16) &&
                   rows_allow(dy, dy_sb, dy_st, es, 16) ? 16 : in ? 4 : 0;
    scan_launch<true>(p, dtype, W, cb, s);
    if (int e = launch_status("gated_scan_bwd_kernel")) return e;
  } else if (dh0 && B > 0) {  // no steps: the gradient passes through
    const cudaError_t e = dh_last ? cudaMemcpyAsync(dh0, dh_last, (size_t)B * ds * 4, cudaMemcpyDeviceToDevice, s)
                                  : cudaMemsetAsync(dh0, 0, (size_t)B * ds * 4, s);
    if (e != cudaSuccess) return fail((int)e, "gated_scan_bwd: %s", cudaGetErrorString(e));
  }
  gated_scan_dA_kernel<<<(unsigned)((ds + 31) / 32), 1024, 0, s>>>(p.dA_part, (int64_t)p.NT * B, p.nch * p.CW, (int)ds,
                                                                  A_log, p.a_bf16, dA_log);
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
