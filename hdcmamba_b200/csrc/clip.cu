// The norm over all gradients of a model, and the gradients scaled to it:
//   norm = sqrt(sum over all tensors and elements of g^2),  out = g * min(1, max_norm / (norm + 1e-6)).
//
// Bound by traffic: the gradients are read for the norm, and read and written to be scaled.  All tensors
// are cut into pieces of 16 KB; a kernel's CTAs share the pieces, whatever tensor they belong to, so a
// launch serves up to kTensors tensors of mixed sizes and types.  The table of tensors is a kernel
// argument: nothing is copied to the device beforehand, and a captured call needs no memory of the
// host's.  Gradients that stay as they are, in place, the second kernel does not touch.
// 76.5 M bf16 gradients into other buffers: 76 us for 459 MB, 6.0 TB/s, in place 78 us; 190 M 190 us.  Reads beside
// writes go no faster whatever the number of CTAs (2 to 6 per SM), the size of a piece or a second piece in flight: what
// helps is less traffic, so the second kernel walks the pieces backwards and finds the last 64 MB in L2, which the first
// one loads the ordinary way and all others as the first to let go (86 and 211 us without; 32, 80 and 100 MB are no better).
// Asking L2 to keep the 64 MB above all else gains nothing here (77, 80 and 192 us), and where the second kernel has
// nothing to read it would bind half of L2 for what comes later: a kernel over 100 MB that are in L2 35 us for 31.
// Sums: a thread adds the squares of a piece's 16 or 32 elements in fp32, and those sums in 64 bits; the CTAs'
// sums are added in a fixed order.  Where squares leave fp32's range (|g| above 1e18 or all below 1e-16)
// a thread takes its elements again in 64 bits.
#include <algorithm>
#include <memory>

#include "common.cuh"
#include "vec.cuh"

namespace hdc {

constexpr int kTensors = 512, kThreads = 256, kVecs = 4, kPerSm = 4, kCtas = 148 * kPerSm;
constexpr int kKeep = 4096;  // the last pieces, 64 MB, that stay in L2 from the first kernel to the second
template <typename T> constexpr int kPiece = kThreads * kVecs * Vec<T>::N;  // elements: 16 KB

struct ClipTable {
  const void* in[kTensors];
  void* out[kTensors];
  int64_t n[kTensors];
  int first[kTensors + 1];  // a tensor's first piece; behind the last tensor: the number of pieces
  uint8_t bf16[kTensors];
  int tensors;
};

// elements before the first 16-byte boundary: the first piece has them beside its own
template <typename T> __host__ __device__ inline int64_t lead(const void* p, int64_t n) {
  const int64_t k = (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int64_t)sizeof(T);
  return n < k ? n : k;
}

// The pieces of a CTA, every gridDim-th (the CTAs together read one stretch of memory), forwards or backwards, and
// the tensor of each.
struct Walk {
  const ClipTable& t;
  int i, step, k, pieces;
  __device__ __forceinline__ Walk(const ClipTable& table, bool backwards) : t(table), pieces(table.first[table.tensors]) {
    step = backwards ? -(int)gridDim.x : (int)gridDim.x;
    i = backwards ? pieces - 1 - (int)blockIdx.x : (int)blockIdx.x;
    k = backwards ? t.tensors - 1 : 0;
    find();
  }
  __device__ __forceinline__ bool more() const { return i >= 0 && i < pieces; }
  __device__ __forceinline__ void find() {
    if (!more()) return;
    while (i >= t.first[k + 1]) ++k;
    while (i < t.first[k]) --k;
  }
  __device__ __forceinline__ void next() {
    i += step;
    find();
  }
};
struct Place {
  const char* in;  // the piece's first 16-byte vector
  char* out;       // the same element of the output
  int vecs;        // whole vectors; behind the last piece: -1
  int head, tail;  // single elements before the first vector (in a tensor's first piece) and behind the last
  int bf16;
  bool together;   // in and out reach 16-byte boundaries together
  __device__ __forceinline__ explicit Place(const Walk& w) : vecs(-1) {
    if (!w.more()) return;
    bf16 = w.t.bf16[w.k];
    const int es = bf16 ? 2 : 4, per = bf16 ? kPiece<__nv_bfloat16> : kPiece<float>;
    const void* p = w.t.in[w.k];
    const int64_t n = w.t.n[w.k];
    const int piece = w.i - w.t.first[w.k];
    const int64_t k = bf16 ? lead<__nv_bfloat16>(p, n) : lead<float>(p, n), begin = k + (int64_t)piece * per;
    const int count = (int)min((int64_t)per, n - begin);
    in = static_cast<const char*>(p) + begin * es;
    out = static_cast<char*>(w.t.out[w.k]) + begin * es;
    vecs = count * es / 16;
    head = piece == 0 ? (int)k : 0;
    tail = count - vecs * (16 / es);
    together = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  }
  // the element that a thread has beside the vectors, as a distance in elements from `in`, or no = kNone
  static constexpr int kNone = 1 << 30;
  __device__ __forceinline__ int single() const {
    const int i = (int)threadIdx.x;
    return i < head ? i - head : i < head + tail ? vecs * (bf16 ? 8 : 4) + i - head : kNone;
  }
};

// 16 bytes that L2 keeps or lets go, by the policy.  RO: nothing writes them while the kernel runs; the kernel that
// scales may do so in place, and loads them the ordinary way.
template <bool RO> __device__ __forceinline__ uint4 ldg16_hint(const void* p, uint64_t policy) {
  uint4 r;
  if constexpr (RO) {
    asm volatile("ld.global.nc.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p), "l"(policy));
  } else {
    asm volatile("ld.global.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p), "l"(policy) : "memory");
  }
  return r;
}
// A piece's values in registers; zeros where there are none.
struct Held {
  uint4 w[kVecs];
  float one;
  template <bool RO> __device__ __forceinline__ void load(const Place& p, uint64_t policy) {
    const char* q = p.in + threadIdx.x * 16;
    if (p.vecs == kThreads * kVecs) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) w[i] = ldg16_hint<RO>(q + i * kThreads * 16, policy);
    } else {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        w[i] = make_uint4(0, 0, 0, 0);
        if (i * kThreads + (int)threadIdx.x < p.vecs) w[i] = ldg16_hint<RO>(q + i * kThreads * 16, policy);
      }
    }
    one = 0.f;
    if (p.head + p.tail > 0) {
      const int at = p.single();
      if (at != Place::kNone)
        one = p.bf16 ? to_f(reinterpret_cast<const __nv_bfloat16*>(p.in)[at]) : reinterpret_cast<const float*>(p.in)[at];
    }
  }
};

// x^2 of two values added to two sums
__device__ __forceinline__ void add_squares(uint64_t& s, float x, float y) {
  const uint64_t v = pair_bits(x, y);
  asm("fma.rn.f32x2 %0, %1, %1, %0;" : "+l"(s) : "l"(v));
}
template <typename T> __device__ __forceinline__ double squares(const Held& v) {
  constexpr int V = Vec<T>::N;
  uint64_t s2[2] = {0, 0};
  uint32_t bits = __float_as_uint(v.one);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    float x[V];
    unpack16<T>(v.w[i], x);
#pragma unroll
    for (int j = 0; j < V; j += 2) add_squares(s2[j / 2 & 1], x[j], x[j + 1]);
    bits |= v.w[i].x | v.w[i].y | v.w[i].z | v.w[i].w;
  }
  float a, b, c, d;
  bits_pair(s2[0], a, b);
  bits_pair(s2[1], c, d);
  const float s = fmaf(v.one, v.one, (a + b) + (c + d));
  // all zeros, or squares well inside fp32's range
  if ((s > 1e-32f && s < 3e38f) || (bits & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu)) == 0) return s;
  double e = (double)v.one * v.one;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    float x[V];
    unpack16<T>(v.w[i], x);
#pragma unroll
    for (int j = 0; j < V; ++j) e += (double)x[j] * x[j];
  }
  return e;
}

__device__ __forceinline__ double cta_sum(double v) {
  __shared__ double s[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
  __syncthreads();
  double r = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) r += s[i];
  return r;
}

// The place of the next piece is looked up while a piece's values are on their way.
__global__ void __launch_bounds__(kThreads, kPerSm) grad_squares_kernel(const __grid_constant__ ClipTable t, double* sums,
                                                                        int keep_from) {
  let_next_start();
  double d = 0;
  Walk w(t, false);
  uint64_t stay, go;
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(stay));
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(go));
  for (Place at(w); at.vecs >= 0;) {
    Held v;
    v.load<true>(at, w.i >= keep_from ? stay : go);
    const int bf16 = at.bf16;
    w.next();
    at = Place(w);
    d += bf16 ? squares<__nv_bfloat16>(v) : squares<float>(v);
  }
  d = cta_sum(d);
  if (threadIdx.x == 0) sums[blockIdx.x] = d;
}

// Written values need not stay in L2: what this kernel has not read yet should.
__device__ __forceinline__ void stg16_stream(void* p, const uint4& v) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <typename T> __device__ __forceinline__ void scale_piece(const Held& v, const Place& p, float by) {
  constexpr int V = Vec<T>::N;
  if (p.head + p.tail > 0) {
    const int at = p.single();
    if (at != Place::kNone) reinterpret_cast<T*>(p.out)[at] = from_f<T>(v.one * by);
  }
  char* q = p.out + threadIdx.x * 16;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    if (i * kThreads + (int)threadIdx.x >= p.vecs) continue;
    float x[V];
    unpack16<T>(v.w[i], x);
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      uint64_t r;
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(x[j], x[j + 1])), "l"(pair_bits(by, by)));
      bits_pair(r, x[j], x[j + 1]);
    }
    if (p.together) {
      stg16_stream(q + i * kThreads * 16, pack16<T>(x));
    } else {
      T* o = reinterpret_cast<T*>(q + i * kThreads * 16);
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = from_f<T>(x[j]);
    }
  }
}

__global__ void __launch_bounds__(kThreads, kPerSm) grad_scale_kernel(const __grid_constant__ ClipTable t, const double* sums,
                                                                      int n_sums, float max_norm, float* norm_out) {
  wait_for_previous();
  double d = 0;
  for (int i = threadIdx.x; i < n_sums; i += kThreads) d += sums[i];
  const double norm = sqrt(cta_sum(d));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double c = (double)max_norm / (norm + 1e-6);
  const float by = c >= 1.0 ? 1.f : (float)c;  // NaN stays
  uint64_t go;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(go));
  Walk w(t, true);
  for (Place at(w); at.vecs >= 0;) {
    const Place p = at;
    const bool skip = by == 1.f && p.in == p.out;  // it stays as it is
    Held v;
    if (!skip) v.load<false>(p, go);
    w.next();
    at = Place(w);
    if (!skip) p.bf16 ? scale_piece<__nv_bfloat16>(v, p, by) : scale_piece<float>(v, p, by);
  }
}

static int64_t pieces_of(const void* p, int64_t n, int dtype) {
  const bool f32 = dtype == HDC_F32;
  const int64_t m = n - (f32 ? lead<float>(p, n) : lead<__nv_bfloat16>(p, n)), per = f32 ? kPiece<float> : kPiece<__nv_bfloat16>;
  return m <= per ? 1 : (m + per - 1) / per;
}

struct Span { uintptr_t begin, end; int tensor, out; };

// every output lies apart from the other outputs and from the gradients, but may be its own gradient
static int clip_overlaps(int64_t n, const int* dtypes, const void* const* grads, void* const* outs,
                         const int64_t* numels) {
  std::unique_ptr<Span[]> s(new Span[2 * n]);
  int64_t m = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (numels[i] == 0) continue;
    const uintptr_t bytes = (uintptr_t)numels[i] * (dtypes[i] == HDC_F32 ? 4 : 2);
    const uintptr_t g = reinterpret_cast<uintptr_t>(grads[i]), o = reinterpret_cast<uintptr_t>(outs[i]);
    s[m++] = {o, o + bytes, (int)i, 1};
    if (g != o) s[m++] = {g, g + bytes, (int)i, 0};
  }
  std::sort(s.get(), s.get() + m, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t out_end = 0, any_end = 0;
  for (int64_t i = 0; i < m; ++i) {
    if (s[i].begin < out_end || (s[i].out && s[i].begin < any_end))
      return fail(HDC_E_SHAPE, "clip_grads: output %d overlaps another output or a gradient", s[i].tensor);
    if (s[i].out && s[i].end > out_end) out_end = s[i].end;
    if (s[i].end > any_end) any_end = s[i].end;
  }
  return HDC_OK;
}

static int64_t clip_groups(int64_t n) { return n < 1 ? 1 : (n + kTensors - 1) / kTensors; }

static int clip(int64_t n, const int* dtypes, const void* const* grads, void* const* outs, const int64_t* numels,
                float max_norm, float* norm, void* workspace, size_t workspace_bytes, cudaStream_t s) {
  if (n < 0 || n > (1 << 20)) return fail(HDC_E_SHAPE, "clip_grads: %lld tensors (0 to 2^20)", (long long)n);
  if (!norm || !workspace || (n > 0 && (!dtypes || !grads || !numels))) return fail(HDC_E_NULL, "clip_grads: null pointer");
  if (outs && !(max_norm >= 0.f)) return fail(HDC_E_SHAPE, "clip_grads: max_norm=%g", (double)max_norm);
  const int64_t groups = clip_groups(n);
  if (workspace_bytes < (size_t)groups * kCtas * 8)
    return fail(HDC_E_WORKSPACE, "clip_grads: workspace of %zu bytes, %zu needed", workspace_bytes, (size_t)groups * kCtas * 8);
  if (!aligned16(workspace) || (reinterpret_cast<uintptr_t>(norm) & 3) != 0)
    return fail(HDC_E_ALIGN, "clip_grads: the workspace or norm is not aligned");
  for (int64_t i = 0; i < n; ++i) {
    if (dtypes[i] != HDC_F32 && dtypes[i] != HDC_BF16) return fail(HDC_E_DTYPE, "clip_grads: tensor %lld: dtype %d", (long long)i, dtypes[i]);
    const uintptr_t mask = dtypes[i] == HDC_F32 ? 3 : 1;
    if (numels[i] < 0 || numels[i] > (int64_t(1) << 40)) return fail(HDC_E_SHAPE, "clip_grads: tensor %lld has %lld elements", (long long)i, (long long)numels[i]);
    if (numels[i] > 0 && (!grads[i] || (outs && !outs[i]))) return fail(HDC_E_NULL, "clip_grads: tensor %lld is null", (long long)i);
    if ((reinterpret_cast<uintptr_t>(grads[i]) & mask) || (outs && (reinterpret_cast<uintptr_t>(outs[i]) & mask)))
      return fail(HDC_E_ALIGN, "clip_grads: tensor %lld is not aligned to its type", (long long)i);
  }
  if (outs)
    if (int e = clip_overlaps(n, dtypes, grads, outs, numels)) return e;
  auto sums = static_cast<double*>(workspace);
  std::unique_ptr<ClipTable> t(new ClipTable);
  int used = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t g = 0; g < groups; ++g) {
      t->tensors = 0;
      int64_t pieces = 0;
      for (int64_t i = g * kTensors; i < n && i < (g + 1) * kTensors; ++i) {
        if (numels[i] == 0) continue;
        const int k = t->tensors++;
        t->in[k] = grads[i];
        t->out[k] = outs ? outs[i] : nullptr;
        t->n[k] = numels[i];
        t->bf16[k] = dtypes[i] == HDC_BF16;
        t->first[k] = (int)pieces;
        pieces += pieces_of(grads[i], numels[i], dtypes[i]);
        if (pieces >= (int64_t(1) << 30)) return fail(HDC_E_SHAPE, "clip_grads: too many elements");
      }
      t->first[t->tensors] = (int)pieces;
      const int grid = (int)std::min<int64_t>(kCtas, pieces);
      if (pass == 0) {
        if (grid == 0) continue;
        const int keep_from = outs && g + 1 == groups ? (int)pieces - kKeep : (int)pieces;
        grad_squares_kernel<<<grid, kThreads, 0, s>>>(*t, sums + used, keep_from);
        used += grid;
        if (int e = launch_status("grad_squares_kernel")) return e;
      } else if (g == 0 || (grid > 0 && outs)) {
        if (!outs) t->tensors = t->first[0] = 0;
        launch_dependent(grad_scale_kernel, dim3(outs && grid > 0 ? grid : 1), kThreads, 0, s, *t, static_cast<const double*>(sums),
                         used, max_norm, g == 0 ? norm : nullptr);
        if (int e = launch_status("grad_scale_kernel")) return e;
      }
    }
  }
  return HDC_OK;
}

}  // namespace hdc

using namespace hdc;

extern "C" size_t hdc_clip_grads_workspace_bytes(int64_t n) { return (size_t)clip_groups(n) * kCtas * 8; }

extern "C" int hdc_clip_grads(int64_t n, const int* dtypes, const void* const* grads, void* const* outs,
                              const int64_t* numels, float max_norm, float* norm, void* workspace,
                              size_t workspace_bytes, hdc_stream_t stream) {
  try {
    return clip(n, dtypes, grads, outs, numels, max_norm, norm, workspace, workspace_bytes,
                reinterpret_cast<cudaStream_t>(stream));
  } catch (...) {
    return fail(HDC_E_SHAPE, "clip_grads: out of host memory");
  }
}
