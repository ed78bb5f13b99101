// The norm over all gradients of a model, and the gradients scaled to it:
//   norm = sqrt(sum over all tensors and elements of g^2),  out = g * min(1, max_norm / (norm + 1e-6)).
//
// Bound by traffic: the gradients are read for the norm, and read and written to be scaled.  All tensors
// are cut into pieces of kPiece elements; a kernel's CTAs take the pieces in turn, whatever tensor they
// belong to, so a launch serves up to kTensors tensors of mixed sizes and types.  The table of tensors
// is a kernel argument: nothing is copied to the device beforehand, and a captured call needs no memory
// of the host's.  The second kernel walks the pieces backwards, since L2 (126 MB) still holds the ones
// that were read last; gradients that stay as they are, in place, it does not touch.
// Sums: a thread adds the squares of kPiece / 256 elements in fp32, and those sums in 64 bits; the CTAs'
// sums are added in a fixed order.  Where squares leave fp32's range (|g| above 1e18 or all below 1e-16)
// a thread takes its elements again in 64 bits.
#include <algorithm>
#include <memory>

#include "common.cuh"

namespace hdc {

constexpr int kTensors = 512, kThreads = 256, kPiece = 8192, kCtas = 148 * 4;

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

// One piece as a thread sees it: 16-byte vectors, then at most two single elements (before the first
// vector of the tensor's first piece, and behind the last one).
template <typename T> struct Piece {
  static constexpr int V = Vec<T>::N, kVecs = kPiece / V / kThreads;
  const T* p;
  int64_t begin, end, head, tail;  // head, tail: a single element's index, or -1
  int vecs;
  __device__ __forceinline__ Piece(const void* q, int64_t n, int piece) {
    p = static_cast<const T*>(q);
    const int64_t k = lead<T>(q, n);
    begin = k + (int64_t)piece * kPiece;
    end = min(n, begin + kPiece);
    vecs = (int)((end - begin) / V);
    head = piece == 0 && (int)threadIdx.x < k ? (int)threadIdx.x : -1;
    tail = begin + (int64_t)vecs * V + threadIdx.x;
    if (tail >= end) tail = -1;
  }
  // element index of vector i, or -1
  __device__ __forceinline__ int64_t at(int i) const {
    const int v = i * kThreads + threadIdx.x;
    return v < vecs ? begin + (int64_t)v * V : -1;
  }
};

__device__ __forceinline__ int tensor_of(const ClipTable& t, int piece) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int m = (lo + hi + 1) / 2;
    if (t.first[m] <= piece) lo = m;
    else hi = m - 1;
  }
  return lo;
}

template <typename T> __device__ __forceinline__ double squares(const void* q, int64_t n, int piece) {
  using P = Piece<T>;
  const P p(q, n, piece);
  uint4 w[P::kVecs];
#pragma unroll
  for (int i = 0; i < P::kVecs; ++i) w[i] = ldg16_pred(p.at(i) < 0 ? p.p : p.p + p.at(i), p.at(i) >= 0);
  const float h = p.head >= 0 ? to_f(p.p[p.head]) : 0.f, t = p.tail >= 0 ? to_f(p.p[p.tail]) : 0.f;
  float s = fmaf(h, h, t * t), most = fmaxf(fabsf(h), fabsf(t));
#pragma unroll
  for (int i = 0; i < P::kVecs; ++i) {
    float x[P::V];
    unpack16<T>(w[i], x);
#pragma unroll
    for (int j = 0; j < P::V; ++j) {
      s = fmaf(x[j], x[j], s);
      most = fmaxf(most, fabsf(x[j]));
    }
  }
  if (most < 1e18f && (s > 1e-32f || most == 0.f) && s == s) return s;
  double d = (double)h * h + (double)t * t;
#pragma unroll
  for (int i = 0; i < P::kVecs; ++i) {
    float x[P::V];
    unpack16<T>(w[i], x);
#pragma unroll
    for (int j = 0; j < P::V; ++j) d += (double)x[j] * x[j];
  }
  return d;
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

__global__ void __launch_bounds__(kThreads) grad_squares_kernel(const __grid_constant__ ClipTable t, double* sums) {
  double d = 0;
  const int pieces = t.first[t.tensors];
  for (int i = blockIdx.x; i < pieces; i += gridDim.x) {
    const int k = tensor_of(t, i);
    d += t.bf16[k] ? squares<__nv_bfloat16>(t.in[k], t.n[k], i - t.first[k])
                   : squares<float>(t.in[k], t.n[k], i - t.first[k]);
  }
  d = cta_sum(d);
  if (threadIdx.x == 0) sums[blockIdx.x] = d;
}

template <typename T> __device__ __forceinline__ void scale_piece(const void* q, void* out, int64_t n, int piece, float by) {
  using P = Piece<T>;
  const P p(q, n, piece);
  T* o = static_cast<T*>(out);
  if (((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(out)) & 15) != 0) {
    // the two do not reach 16-byte boundaries together
    const int64_t b = piece == 0 ? 0 : p.begin;
    for (int64_t i = b + threadIdx.x; i < p.end; i += kThreads) o[i] = from_f<T>(to_f(p.p[i]) * by);
    return;
  }
  uint4 w[P::kVecs];
#pragma unroll
  for (int i = 0; i < P::kVecs; ++i)
    if (p.at(i) >= 0) w[i] = *reinterpret_cast<const uint4*>(p.p + p.at(i));
  if (p.head >= 0) o[p.head] = from_f<T>(to_f(p.p[p.head]) * by);
  if (p.tail >= 0) o[p.tail] = from_f<T>(to_f(p.p[p.tail]) * by);
#pragma unroll
  for (int i = 0; i < P::kVecs; ++i) {
    if (p.at(i) < 0) continue;
    float x[P::V];
    unpack16<T>(w[i], x);
#pragma unroll
    for (int j = 0; j < P::V; ++j) x[j] *= by;
    stg16(o + p.at(i), pack16<T>(x));
  }
}

__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ ClipTable t, const double* sums,
                                                              int n_sums, float max_norm, float* norm_out) {
  double d = 0;
  for (int i = threadIdx.x; i < n_sums; i += kThreads) d += sums[i];
  const double norm = sqrt(cta_sum(d));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double c = (double)max_norm / (norm + 1e-6);
  const float by = c >= 1.0 ? 1.f : (float)c;  // NaN stays
  const int pieces = t.first[t.tensors];
  for (int j = blockIdx.x; j < pieces; j += gridDim.x) {
    const int i = pieces - 1 - j, k = tensor_of(t, i);
    if (by == 1.f && t.in[k] == t.out[k]) continue;
    if (t.bf16[k]) scale_piece<__nv_bfloat16>(t.in[k], t.out[k], t.n[k], i - t.first[k], by);
    else scale_piece<float>(t.in[k], t.out[k], t.n[k], i - t.first[k], by);
  }
}

static int64_t pieces_of(const void* p, int64_t n, int dtype) {
  const int64_t m = n - (dtype == HDC_F32 ? lead<float>(p, n) : lead<__nv_bfloat16>(p, n));
  return m <= kPiece ? 1 : (m + kPiece - 1) / kPiece;
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
        grad_squares_kernel<<<grid, kThreads, 0, s>>>(*t, sums + used);
        used += grid;
        if (int e = launch_status("grad_squares_kernel")) return e;
      } else if (g == 0 || (grid > 0 && outs)) {
        if (!outs) t->tensors = t->first[0] = 0;
        grad_scale_kernel<<<outs && grid > 0 ? grid : 1, kThreads, 0, s>>>(*t, sums, used, max_norm, g == 0 ? norm : nullptr);
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
