// Token embedding: y_n = scale * table[id_n], and its gradient dtable[v] = scale * sum over id_n = v of dy_n.
//
// Lookup.  Rows are copied 16 bytes a thread, kLoads of them in flight, with no staging: the kernel is
// bound by the table's and the output's traffic.
//
// Gradient.  Tokens are sorted by id, stably (least significant digit first, at most 9 bits a pass), so
// that each row's sum is taken in the tokens' own order and the result does not depend on timing: no
// floating-point atomics.  Rows and sorted tokens then form one merged list (a row's tokens, then its
// end), of which every warp takes an equal part, so that neither a frequent id nor a wide table leaves
// warps idle: a token costs one row read, a row's end one row written (zeros where no token has it).
// A row cut by a part's border leaves fp32 partial sums that a last kernel adds in the parts' order.
#include "tc.cuh"
#include "vec.cuh"

namespace hdc {

constexpr int kBadId = 71;  // hdc_device_error: an id outside the table

template <typename I>
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t n) {
  return static_cast<const I*>(ids)[n];
}

// ---------------------------------------------------------------- lookup
constexpr int kLoads = 4;

// nv: vectors of V elements of a row.  Block i takes vectors [i * 256 * kLoads, ...) of all rows' vectors.
template <typename T, typename I, int V>
__global__ void __launch_bounds__(256) embedding_kernel(const void* ids, const T* table, int64_t table_st, T* y,
                                                        int64_t y_st, int64_t N, int64_t rows, int nv, float scale) {
  const int64_t first = (int64_t)blockIdx.x * 256 * kLoads;
  const int64_t n0 = first / nv;
  const unsigned off = (unsigned)(first - n0 * nv) + threadIdx.x;
  uint4 w[kLoads];
  T e[kLoads];
  int64_t id[kLoads];
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const unsigned k = off + u * 256;
    const int64_t n = n0 + k / (unsigned)nv;
    id[u] = n < N ? id_at<I>(ids, n) : -1;
    if (n < N && (id[u] < 0 || id[u] >= rows)) atomicCAS(&g_dev_error, 0, kBadId);
  }
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const unsigned c = (off + u * 256) % (unsigned)nv;
    const bool ok = id[u] >= 0 && id[u] < rows;
    const T* src = table + id[u] * table_st + (int64_t)c * V;
    if constexpr (V == 1) e[u] = ok ? *src : from_f<T>(0.f);
    else w[u] = ldg16_pred(ok ? src : table, ok);
  }
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const unsigned k = off + u * 256, c = k % (unsigned)nv;
    const int64_t n = n0 + k / (unsigned)nv;
    if (n >= N) continue;
    const float by = id[u] >= 0 && id[u] < rows ? scale : __int_as_float(0x7fffffff);
    T* dst = y + n * y_st + (int64_t)c * V;
    if constexpr (V == 1) {
      *dst = from_f<T>(by * to_f(e[u]));
    } else {
      float f[V];
      unpack16<T>(w[u], f);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= by;
      stg16(dst, pack16<T>(f));
    }
  }
}

// ---------------------------------------------------------------- sort by id
constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32, kMaxBins = 512;
constexpr int kTileLeast = 1024, kMostTiles = 128;

struct SortPlan {
  int passes, bits;      // digit passes and bits of a digit
  int tiles;             // tiles of `tile` tokens, a multiple of 256
  int64_t tile;
};

// the id that sorts a token: `rows` (behind all) where it takes no part in the gradient
template <typename I>
__device__ __forceinline__ unsigned sort_key(const void* ids, int64_t n, int64_t rows, int64_t skip) {
  const int64_t id = id_at<I>(ids, n);
  if (id < 0 || id >= rows) {
    atomicCAS(&g_dev_error, 0, kBadId);
    return (unsigned)rows;
  }
  return id == skip ? (unsigned)rows : (unsigned)id;
}

// Counts of the first digit of each tile, and zeros in the later digits' tables ([pass][tile][bin]).
template <typename I>
__global__ void __launch_bounds__(kSortThreads) embedding_count_kernel(const void* ids, int64_t N, int64_t rows,
                                                                       int64_t skip, SortPlan p, unsigned* counts) {
  __shared__ unsigned c[kMaxBins];
  const int bins = 1 << p.bits;
  for (int i = threadIdx.x; i < bins; i += kSortThreads) c[i] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * p.tile, end = min(N, begin + p.tile);
  for (int64_t n = begin + threadIdx.x; n < end; n += kSortThreads)
    atomicAdd(&c[sort_key<I>(ids, n, rows, skip) & (bins - 1)], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += kSortThreads) {
    counts[(int64_t)blockIdx.x * bins + i] = c[i];
    for (int k = 1; k < p.passes; ++k) counts[((int64_t)k * p.tiles + blockIdx.x) * bins + i] = 0;
  }
}

// One digit's pass: (key, token) pairs move to their place by (digit, tile, place in the tile).  A tile's
// place for each digit follows from all tiles' counts, which its CTA adds up itself.
template <typename I>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const void* ids, const uint2* from, uint2* to,
                                                                      int64_t N, int64_t rows, int64_t skip,
                                                                      SortPlan p, int pass, unsigned* counts) {
  __shared__ unsigned base[kMaxBins];                 // where the next of each digit goes
  __shared__ unsigned part[kSortWarps][kMaxBins];     // a round's counts, warp by warp
  __shared__ unsigned sums[kSortWarps];
  const int bins = 1 << p.bits, shift = pass * p.bits;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const unsigned* table = counts + (int64_t)pass * p.tiles * bins;
  unsigned* next = pass + 1 < p.passes ? counts + (int64_t)(pass + 1) * p.tiles * bins : nullptr;
  // digits 2 * thread and 2 * thread + 1: the tokens of all tiles, and those of the tiles before this one
  unsigned all[2] = {0, 0}, before[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int d = threadIdx.x * 2 + e;
    if (d >= bins) continue;
#pragma unroll 8
    for (int t = 0; t < p.tiles; ++t) {
      const unsigned c = table[(int64_t)t * bins + d];
      all[e] += c;
      before[e] += t < (int)blockIdx.x ? c : 0;
    }
  }
  unsigned x = all[0] + all[1];  // running sum over the digits
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  unsigned lower = x - all[0] - all[1];
  for (int w = 0; w < warp; ++w) lower += sums[w];
  if (threadIdx.x * 2 < bins) {
    base[threadIdx.x * 2] = lower + before[0];
    base[threadIdx.x * 2 + 1] = lower + all[0] + before[1];
  }
  const int64_t begin = blockIdx.x * p.tile, end = min(N, begin + p.tile);
  for (int64_t n0 = begin; n0 < end; n0 += kSortThreads) {
    for (int i = threadIdx.x; i < bins * kSortWarps; i += kSortThreads) part[i / bins][i % bins] = 0;
    const int64_t n = n0 + threadIdx.x;
    uint2 e = make_uint2(0, 0);
    if (n < end) e = pass == 0 ? make_uint2(sort_key<I>(ids, n, rows, skip), (unsigned)n) : from[n];
    const int d = n < end ? (int)((e.x >> shift) & (unsigned)(bins - 1)) : bins;  // bins: no token
    const unsigned same = __match_any_sync(0xffffffffu, d);
    const int rank = __popc(same & ((1u << lane) - 1));
    __syncthreads();
    if (d < bins && rank == 0) part[warp][d] = __popc(same);
    __syncthreads();
    if (d < bins) {
      unsigned at = base[d] + rank;
      for (int w = 0; w < warp; ++w) at += part[w][d];
      to[at] = e;
      if (next) atomicAdd(&next[(int64_t)(at / p.tile) * bins + ((e.x >> (shift + p.bits)) & (unsigned)(bins - 1))], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += kSortThreads) {
      unsigned c = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) c += part[w][i];
      base[i] += c;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- sums
// Part u of the merged list: items [u * items, (u + 1) * items).  Partial sums [parts][D] fp32.
struct SumPlan {
  int64_t items, parts;
};

// tokens among the first d items: the most t with key[t - 1] <= d - t
__device__ __forceinline__ int64_t merge_split(const uint2* sorted, int64_t N, int64_t rows, int64_t d) {
  int64_t lo = d > rows ? d - rows : 0, hi = d < N ? d : N;
  while (lo < hi) {
    const int64_t t = (lo + hi + 1) / 2;
    if ((int64_t)sorted[t - 1].x <= d - t) lo = t;
    else hi = t - 1;
  }
  return lo;
}

// V consecutive elements of a lane (V = 1: 8 elements 32 apart)
template <typename T, bool VEC> struct Cols {
  static constexpr int N = VEC ? Vec<T>::N : 8;
  static constexpr int kWarp = 32 * N;  // columns of a warp
};
template <typename T, bool VEC>
__device__ __forceinline__ void col_load(const T* row, int c0, int lane, int D, float* f) {
  if constexpr (VEC) {
    const int c = c0 + lane * Vec<T>::N;
    unpack16<T>(ldg16_pred(row + (c < D ? c : 0), c < D), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + i * 32 + lane;
      f[i] = c < D ? to_f(row[c]) : 0.f;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void col_store(T* row, int c0, int lane, int D, const float* f) {
  if constexpr (VEC) {
    const int c = c0 + lane * Vec<T>::N;
    if (c < D) stg16(row + c, pack16<T>(f));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + i * 32 + lane;
      if (c < D) row[c] = from_f<T>(f[i]);
    }
  }
}
// partial sums: a lane's elements in its own order, [part][column block][lane][N]
template <int N>
__device__ __forceinline__ float* part_at(float* p, int64_t u, int lane) {
  return p + ((u * gridDim.y + blockIdx.y) * 32 + lane) * N;
}

constexpr int kSumWarps = 4, kRowsAhead = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kSumWarps * 32) embedding_sum_kernel(const uint2* sorted, const T* dy, int64_t dy_st,
                                                                       T* dtable, int64_t d_st, int64_t N,
                                                                       int64_t rows, int D, float scale, SumPlan p,
                                                                       int* heads, int* tails, float* head_sums,
                                                                       float* tail_sums) {
  using C = Cols<T, VEC>;
  const int lane = threadIdx.x % 32, c0 = blockIdx.y * C::kWarp;
  const int64_t u = (int64_t)blockIdx.x * kSumWarps + threadIdx.x / 32;
  if (u >= p.parts) return;
  const int64_t d0 = u * p.items, d1 = min(d0 + p.items, rows + N);
  int64_t t = merge_split(sorted, N, rows, d0);
  const int64_t t_end = merge_split(sorted, N, rows, d1), r_end = d1 - t_end;
  int64_t r = d0 - t;
  // the first row began in an earlier part
  bool begun = t > 0 && (int64_t)sorted[t - 1].x == r;
  int head = -1, tail = -1;
  float acc[C::N];
#pragma unroll
  for (int i = 0; i < C::N; ++i) acc[i] = 0.f;
  bool any = false;
  while (r < rows) {  // behind the last row: the tokens that take no part
    // a window of tokens: those of row r are the first k of it
    const int64_t m = t + lane;
    const uint2 e = m < t_end ? sorted[m] : make_uint2(0xffffffffu, 0);
    const unsigned mine = __ballot_sync(0xffffffffu, m < t_end && (int64_t)e.x == r);
    const int k = __popc(mine);
    for (int j = 0; j < k; j += kRowsAhead) {
      float f[kRowsAhead][C::N];
#pragma unroll
      for (int a = 0; a < kRowsAhead; ++a) {
        const unsigned n = __shfl_sync(0xffffffffu, e.y, min(j + a, k - 1));
        if (j + a < k) col_load<T, VEC>(dy + (int64_t)n * dy_st, c0, lane, D, f[a]);
      }
#pragma unroll
      for (int a = 0; a < kRowsAhead; ++a)
        if (j + a < k)
#pragma unroll
          for (int i = 0; i < C::N; ++i) acc[i] += f[a][i];
    }
    t += k;
    any = any || k > 0;
    if (k == 32) continue;  // the row may go on
    if (r >= r_end) break;
    if (begun) {
      head = (int)r;
#pragma unroll
      for (int i = 0; i < C::N; ++i) part_at<C::N>(head_sums, u, lane)[i] = acc[i];
    } else {
#pragma unroll
      for (int i = 0; i < C::N; ++i) acc[i] *= scale;
      col_store<T, VEC>(dtable + r * d_st, c0, lane, D, acc);
    }
#pragma unroll
    for (int i = 0; i < C::N; ++i) acc[i] = 0.f;
    begun = any = false;
    ++r;
  }
  if (r < rows && (any || begun)) {  // the row goes on in the next part
    tail = (int)r;
#pragma unroll
    for (int i = 0; i < C::N; ++i) part_at<C::N>(tail_sums, u, lane)[i] = acc[i];
  }
  if (blockIdx.y == 0 && lane == 0) {
    heads[u] = head;
    tails[u] = begun && tail >= 0 ? tail | (1 << 31) : tail;  // sign: the row began in an earlier part
  }
}

// Rows cut by the parts' borders: where a part ended such a row, the parts before it that hold the row's
// beginning are added in order (8 warps take every eighth, and their sums are added in order), then its own.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) embedding_cut_kernel(T* dtable, int64_t d_st, int D, float scale, int64_t parts,
                                                            const int* heads, const int* tails, float* head_sums,
                                                            float* tail_sums) {
  using C = Cols<T, VEC>;
  __shared__ float s[8][32][C::N];
  const int64_t u = blockIdx.x;
  const int head = heads[u];
  if (head < 0) return;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int64_t first = u - 1;  // the part in which the row began
  for (int64_t f0 = u - 1;; f0 -= 32) {
    const int64_t f = f0 - lane;
    const bool through = f >= 0 && tails[f] < -1;
    const unsigned m = __ballot_sync(0xffffffffu, !through);
    if (m != 0) {
      first = f0 - (__ffs(m) - 1);
      break;
    }
  }
  float acc[C::N];
#pragma unroll
  for (int i = 0; i < C::N; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int64_t f = first + warp; f < u; f += 8) {
    const float* q = part_at<C::N>(tail_sums, f, lane);
#pragma unroll
    for (int i = 0; i < C::N; ++i) acc[i] += q[i];
  }
#pragma unroll
  for (int i = 0; i < C::N; ++i) s[warp][lane][i] = acc[i];
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int i = 0; i < C::N; ++i) {
    for (int w = 1; w < 8; ++w) acc[i] += s[w][lane][i];
    acc[i] = scale * (acc[i] + part_at<C::N>(head_sums, u, lane)[i]);
  }
  col_store<T, VEC>(dtable + head * d_st, blockIdx.y * C::kWarp, lane, D, acc);
}

// ---------------------------------------------------------------- plans
static SortPlan sort_plan(int64_t N, int64_t rows) {
  SortPlan p;
  int bits = 1;
  while ((int64_t(1) << bits) <= rows) ++bits;  // the keys are 0 .. rows
  p.passes = (bits + 8) / 9;
  p.bits = (bits + p.passes - 1) / p.passes;
  const int64_t least = (N + kMostTiles - 1) / kMostTiles;
  p.tile = least <= kTileLeast ? kTileLeast : (least + kSortThreads - 1) / kSortThreads * kSortThreads;
  p.tiles = (int)((N + p.tile - 1) / p.tile);
  return p;
}
// Parts for a few waves of warps; at least 16 items, so that a part's search and partial sums stay small
// beside its rows.
static SumPlan sum_plan(int64_t N, int64_t rows) {
  const int64_t total = N + rows;
  int64_t items = (total + 4095) / 4096;
  if (items < 16) items = 16;
  return {items, (total + items - 1) / items};
}
static int64_t padded_cols(int64_t D) { return (D + 255) / 256 * 256; }

static size_t up(size_t n) { return (n + 255) / 256 * 256; }
struct Ws { size_t counts, a, b, heads, tails, head_sums, tail_sums, end; };
static Ws layout(int64_t N, int64_t rows, int64_t D) {
  const SortPlan sp = sort_plan(N, rows);
  const SumPlan su = sum_plan(N, rows);
  Ws w;
  w.counts = 0;
  w.a = up((size_t)sp.passes * sp.tiles * (size_t(1) << sp.bits) * 4);
  w.b = w.a + up((size_t)N * 8);
  w.heads = w.b + up(sp.passes > 1 ? (size_t)N * 8 : 0);
  w.tails = w.heads + up((size_t)su.parts * 4);
  w.head_sums = w.tails + up((size_t)su.parts * 4);
  w.tail_sums = w.head_sums + (size_t)su.parts * padded_cols(D) * 4;
  w.end = w.tail_sums + (size_t)su.parts * padded_cols(D) * 4;
  return w;
}

static int emb_check(const char* what, int dtype, int id_bytes, int64_t N, int64_t rows, int64_t D) {
  if (dtype != HDC_F32 && dtype != HDC_BF16) return fail(HDC_E_DTYPE, "%s: dtype %d", what, dtype);
  if (id_bytes != 4 && id_bytes != 8) return fail(HDC_E_DTYPE, "%s: ids of %d bytes", what, id_bytes);
  if (N < 0 || rows < 1 || D < 1 || N > (int64_t(1) << 30) || rows > (int64_t(1) << 30) || D > 65536)
    return fail(HDC_E_SHAPE, "%s: N=%lld in [0, 2^30], rows=%lld in [1, 2^30], D=%lld in [1, 65536]", what,
                (long long)N, (long long)rows, (long long)D);
  return 0;
}
static bool off(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
// rows of whole 16-byte vectors
static bool vectors(const void* p, int64_t st, int64_t D, int es) {
  return aligned16(p) && st * es % 16 == 0 && D * es % 16 == 0;
}

template <typename T, typename I>
static int lookup(const void* ids, const void* table, int64_t table_st, void* y, int64_t y_st, int64_t N, int64_t rows,
                  int64_t D, float scale, cudaStream_t s) {
  constexpr int V = Vec<T>::N;
  const bool vec = vectors(table, table_st, D, sizeof(T)) && vectors(y, y_st, D, sizeof(T));
  const int nv = (int)(vec ? D / V : D);
  const int64_t blocks = (N * nv + 256 * kLoads - 1) / (256 * kLoads);
  if (blocks >= (int64_t(1) << 31)) return fail(HDC_E_SHAPE, "embedding: N=%lld x D=%lld is too large", (long long)N, (long long)D);
  auto t = static_cast<const T*>(table);
  auto o = static_cast<T*>(y);
  if (vec) embedding_kernel<T, I, V><<<(unsigned)blocks, 256, 0, s>>>(ids, t, table_st, o, y_st, N, rows, nv, scale);
  else embedding_kernel<T, I, 1><<<(unsigned)blocks, 256, 0, s>>>(ids, t, table_st, o, y_st, N, rows, nv, scale);
  return launch_status("embedding_kernel");
}

template <typename T, bool VEC>
static int sums(const uint2* sorted, const void* dy, int64_t dy_st, void* dtable, int64_t d_st, int64_t N, int64_t rows,
                int64_t D, float scale, char* w, const Ws& at, cudaStream_t s) {
  const SumPlan p = sum_plan(N, rows);
  const unsigned cols = (unsigned)((D + Cols<T, VEC>::kWarp - 1) / Cols<T, VEC>::kWarp);
  int *heads = reinterpret_cast<int*>(w + at.heads), *tails = reinterpret_cast<int*>(w + at.tails);
  float *hs = reinterpret_cast<float*>(w + at.head_sums), *ts = reinterpret_cast<float*>(w + at.tail_sums);
  embedding_sum_kernel<T, VEC><<<dim3((unsigned)((p.parts + kSumWarps - 1) / kSumWarps), cols), kSumWarps * 32, 0, s>>>(
      sorted, static_cast<const T*>(dy), dy_st, static_cast<T*>(dtable), d_st, N, rows, (int)D, scale, p, heads, tails,
      hs, ts);
  if (int e = launch_status("embedding_sum_kernel")) return e;
  embedding_cut_kernel<T, VEC><<<dim3((unsigned)p.parts, cols), 256, 0, s>>>(static_cast<T*>(dtable), d_st, (int)D, scale,
                                                                            p.parts, heads, tails, hs, ts);
  return launch_status("embedding_cut_kernel");
}

template <typename T, typename I>
static int gradient(const void* ids, const void* dy, int64_t dy_st, void* dtable, int64_t d_st, int64_t N, int64_t rows,
                    int64_t D, float scale, int64_t skip, char* w, cudaStream_t s) {
  const SortPlan p = sort_plan(N, rows);
  const Ws at = layout(N, rows, D);
  auto counts = reinterpret_cast<unsigned*>(w + at.counts);
  uint2* buf[2] = {reinterpret_cast<uint2*>(w + at.a), reinterpret_cast<uint2*>(w + at.b)};
  if (N > 0) {
    embedding_count_kernel<I><<<p.tiles, kSortThreads, 0, s>>>(ids, N, rows, skip, p, counts);
    if (int e = launch_status("embedding_count_kernel")) return e;
    for (int k = 0; k < p.passes; ++k) {
      embedding_sort_kernel<I><<<p.tiles, kSortThreads, 0, s>>>(ids, buf[(k + 1) % 2], buf[k % 2], N, rows, skip, p, k,
                                                               counts);
      if (int e = launch_status("embedding_sort_kernel")) return e;
    }
  }
  const uint2* sorted = buf[(p.passes + 1) % 2];
  return vectors(dy, dy_st, D, sizeof(T)) && vectors(dtable, d_st, D, sizeof(T))
             ? sums<T, true>(sorted, dy, dy_st, dtable, d_st, N, rows, D, scale, w, at, s)
             : sums<T, false>(sorted, dy, dy_st, dtable, d_st, N, rows, D, scale, w, at, s);
}

}  // namespace hdc

using namespace hdc;

extern "C" int hdc_embedding_fwd(int dtype, const void* ids, int id_bytes, const void* table, int64_t table_st, void* y,
                                 int64_t y_st, float scale, int64_t N, int64_t rows, int64_t D, hdc_stream_t stream) {
  if (int e = emb_check("embedding", dtype, id_bytes, N, rows, D)) return e;
  if (N == 0) return HDC_OK;
  if (!ids || !table || !y) return fail(HDC_E_NULL, "embedding: null pointer");
  const int es = dtype == HDC_F32 ? 4 : 2;
  if (off(table, es) || off(y, es) || off(ids, id_bytes))
    return fail(HDC_E_ALIGN, "embedding: a pointer is not aligned to its type");
  if (N > 1 && y_st < D) return fail(HDC_E_SHAPE, "embedding: rows of y overlap (y_st=%lld)", (long long)y_st);
  auto s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto t, auto i) {
    return lookup<decltype(t), decltype(i)>(ids, table, table_st, y, y_st, N, rows, D, scale, s);
  };
  if (dtype == HDC_F32) return id_bytes == 8 ? go(float(), int64_t()) : go(float(), int32_t());
  return id_bytes == 8 ? go(__nv_bfloat16(), int64_t()) : go(__nv_bfloat16(), int32_t());
}

extern "C" size_t hdc_embedding_bwd_workspace_bytes(int64_t N, int64_t rows, int64_t D) {
  return N < 0 || rows < 1 || D < 1 ? 0 : layout(N, rows, D).end;
}

extern "C" int hdc_embedding_bwd(int dtype, const void* ids, int id_bytes, const void* dy, int64_t dy_st, void* dtable,
                                 int64_t dtable_st, float scale, int64_t skip_id, void* workspace,
                                 size_t workspace_bytes, int64_t N, int64_t rows, int64_t D, hdc_stream_t stream) {
  if (int e = emb_check("embedding_bwd", dtype, id_bytes, N, rows, D)) return e;
  if ((N > 0 && (!ids || !dy)) || !dtable) return fail(HDC_E_NULL, "embedding_bwd: null pointer");
  const int es = dtype == HDC_F32 ? 4 : 2;
  if (off(dy, es) || off(dtable, es) || off(ids, id_bytes))
    return fail(HDC_E_ALIGN, "embedding_bwd: a pointer is not aligned to its type");
  if (rows > 1 && dtable_st < D)
    return fail(HDC_E_SHAPE, "embedding_bwd: rows of dtable overlap (dtable_st=%lld)", (long long)dtable_st);
  const size_t need = layout(N, rows, D).end;
  if (!workspace || workspace_bytes < need)
    return fail(HDC_E_WORKSPACE, "embedding_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  if (!aligned16(workspace)) return fail(HDC_E_ALIGN, "embedding_bwd: the workspace is not 16-byte aligned");
  auto s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto t, auto i) {
    return gradient<decltype(t), decltype(i)>(ids, dy, dy_st, dtable, dtable_st, N, rows, D, scale, skip_id,
                                              static_cast<char*>(workspace), s);
  };
  if (dtype == HDC_F32) return id_bytes == 8 ? go(float(), int64_t()) : go(float(), int32_t());
  return id_bytes == 8 ? go(__nv_bfloat16(), int64_t()) : go(__nv_bfloat16(), int32_t());
}
