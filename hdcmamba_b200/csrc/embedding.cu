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
#include <atomic>

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

// One 16-byte vector (V > 1) or element of an output row from its table row; a bad id gives NaN.
template <typename T, int V> struct Cell {
  uint4 w;
  T e;
  __device__ __forceinline__ void load(const T* src, bool ok) {
    if constexpr (V == 1) e = ok ? *src : from_f<T>(0.f);
    else w = ldg16_pred(src, ok);
  }
  __device__ __forceinline__ void store(T* dst, float by) const {
    if constexpr (V == 1) {
      *dst = from_f<T>(by * to_f(e));
    } else {
      float f[V];
      unpack16<T>(w, f);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= by;
      stg16(dst, pack16<T>(f));
    }
  }
};

// A group of `lanes` lanes (a power of two) copies a row of nv vectors of V elements.  Rows of at most `lanes`
// vectors: a group takes kLoads rows at once; longer ones: kLoads vectors of one row at once.
template <typename T, typename I, int V, bool SHORT>
__global__ void __launch_bounds__(256) embedding_kernel(const void* ids, const T* table, int64_t table_st, T* y,
                                                        int64_t y_st, int64_t N, int64_t rows, int nv, int lanes,
                                                        float scale) {
  const int per_block = 256 / lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  Cell<T, V> cell[kLoads];
  if constexpr (SHORT) {
    const int64_t n0 = (int64_t)blockIdx.x * per_block * kLoads + group;
    int64_t id[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t n = n0 + u * per_block;
      id[u] = n < N ? id_at<I>(ids, n) : 0;
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const bool ok = id[u] >= 0 && id[u] < rows;
      if (!ok) atomicCAS(&g_dev_error, 0, kBadId);
      cell[u].load(table + (ok ? id[u] * table_st : 0) + lane * V, ok && lane < nv && n0 + u * per_block < N);
      id[u] = ok;
    }
    if (lane >= nv) return;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t n = n0 + u * per_block;
      if (n < N) cell[u].store(y + n * y_st + lane * V, id[u] ? scale : __int_as_float(0x7fffffff));
    }
  } else {
    const int64_t n = (int64_t)blockIdx.x * per_block + group;
    if (n >= N) return;
    const int64_t id = id_at<I>(ids, n);
    const bool ok = id >= 0 && id < rows;
    if (!ok) atomicCAS(&g_dev_error, 0, kBadId);
    const T* src = table + (ok ? id * table_st : 0);
    T* dst = y + n * y_st;
    const float by = ok ? scale : __int_as_float(0x7fffffff);
    for (int c0 = lane; c0 < nv; c0 += lanes * kLoads) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int c = c0 + u * lanes;
        cell[u].load(src + (int64_t)(c < nv ? c : 0) * V, ok && c < nv);
      }
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int c = c0 + u * lanes;
        if (c < nv) cell[u].store(dst + (int64_t)c * V, by);
      }
    }
  }
}

// ---------------------------------------------------------------- sort by id
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kMaxBins = 512;
constexpr int kMostTiles = 128;
constexpr int kOneTile = 4096;  // tokens that one CTA sorts in shared memory

struct SortPlan {
  int passes, bits;      // digit passes and bits of a digit
  int tiles;             // tiles of `tile` tokens, a multiple of kSortThreads
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
  let_next_start();
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

// Ranks of a round's tokens (one a thread) among those of the same digit, in the threads' order: a lane's place in
// its warp, the warps before it (part: counts, then running sums), and base[digit], which then moves on.
// d = bins: no token.  Every thread of the CTA calls it.
__device__ __forceinline__ unsigned round_place(int d, int bins, unsigned* base, unsigned short (*part)[kMaxBins]) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i = lane; i < bins / 2; i += 32) reinterpret_cast<unsigned*>(part[warp])[i] = 0;
  __syncwarp();
  const unsigned same = __match_any_sync(0xffffffffu, d);
  const int rank = __popc(same & ((1u << lane) - 1));
  if (d < bins && rank == 0) part[warp][d] = (unsigned short)__popc(same);
  __syncthreads();
  if ((int)threadIdx.x < bins) {
    unsigned sum = base[threadIdx.x];
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const unsigned c = part[w][threadIdx.x];
      part[w][threadIdx.x] = (unsigned short)(sum - base[threadIdx.x]);
      sum += c;
    }
    base[kMaxBins + threadIdx.x] = sum;  // the next round's
  }
  __syncthreads();
  const unsigned at = d < bins ? base[d] + part[warp][d] + rank : 0;
  __syncthreads();
  if ((int)threadIdx.x < bins) base[threadIdx.x] = base[kMaxBins + threadIdx.x];
  return at;  // the caller synchronises before the next round
}

// base[d] = the tokens of lower digits, from counts c of a thread's digit (thread < bins)
__device__ __forceinline__ unsigned lower_digits(unsigned c, unsigned* sums) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  unsigned x = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  unsigned lower = x - c;
  for (int w = 0; w < warp; ++w) lower += sums[w];
  return lower;
}

// One digit's pass: (key, token) pairs move to their place by (digit, tile, place in the tile).  A tile's
// place for each digit follows from all tiles' counts, which its CTA adds up itself.
template <typename I>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const void* ids, const uint2* from, uint2* to,
                                                                      int64_t N, int64_t rows, int64_t skip,
                                                                      SortPlan p, int pass, unsigned* counts) {
  __shared__ unsigned base[2 * kMaxBins], sums[kSortWarps];
  __shared__ __align__(4) unsigned short part[kSortWarps][kMaxBins];
  const int bins = 1 << p.bits, shift = pass * p.bits;
  const unsigned* table = counts + (int64_t)pass * p.tiles * bins;
  unsigned* next = pass + 1 < p.passes ? counts + (int64_t)(pass + 1) * p.tiles * bins : nullptr;
  let_next_start();
  wait_for_previous();
  unsigned all = 0, before = 0;
  if ((int)threadIdx.x < bins) {
#pragma unroll 16
    for (int t = 0; t < p.tiles; ++t) {
      const unsigned c = table[(int64_t)t * bins + threadIdx.x];
      all += c;
      before += t < (int)blockIdx.x ? c : 0;
    }
  }
  const unsigned lower = lower_digits(all, sums);
  if ((int)threadIdx.x < bins) base[threadIdx.x] = lower + before;
  const int64_t begin = blockIdx.x * p.tile, end = min(N, begin + p.tile);
  for (int64_t n0 = begin; n0 < end; n0 += kSortThreads) {
    const int64_t n = n0 + threadIdx.x;
    uint2 e = make_uint2(0, 0);
    if (n < end) e = pass == 0 ? make_uint2(sort_key<I>(ids, n, rows, skip), (unsigned)n) : from[n];
    const int d = n < end ? (int)((e.x >> shift) & (unsigned)(bins - 1)) : bins;
    const unsigned at = round_place(d, bins, base, part);
    if (d < bins) {
      to[at] = e;
      if (next) atomicAdd(&next[(int64_t)(at / p.tile) * bins + ((e.x >> (shift + p.bits)) & (unsigned)(bins - 1))], 1u);
    }
    __syncthreads();
  }
}

// All passes of up to kOneTile tokens by one CTA, in shared memory.
template <typename I>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_one_kernel(const void* ids, uint2* to, int N,
                                                                          int64_t rows, int64_t skip, SortPlan p) {
  constexpr int kRounds = kOneTile / kSortThreads;
  extern __shared__ uint2 sorted[];
  __shared__ unsigned base[2 * kMaxBins], sums[kSortWarps], count[kMaxBins];
  __shared__ __align__(4) unsigned short part[kSortWarps][kMaxBins];
  const int bins = 1 << p.bits;
  let_next_start();
  uint2 e[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int n = i * kSortThreads + threadIdx.x;
    if (n < N) e[i] = make_uint2(sort_key<I>(ids, n, rows, skip), (unsigned)n);
  }
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    for (int i = threadIdx.x; i < bins; i += kSortThreads) count[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRounds; ++i)
      if (i * kSortThreads + (int)threadIdx.x < N) atomicAdd(&count[(e[i].x >> shift) & (unsigned)(bins - 1)], 1u);
    __syncthreads();
    const unsigned lower = lower_digits((int)threadIdx.x < bins ? count[threadIdx.x] : 0, sums);
    if ((int)threadIdx.x < bins) base[threadIdx.x] = lower;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      if (i * kSortThreads >= N) break;
      const int d = i * kSortThreads + (int)threadIdx.x < N ? (int)((e[i].x >> shift) & (unsigned)(bins - 1)) : bins;
      const unsigned at = round_place(d, bins, base, part);
      if (d < bins) sorted[at] = e[i];
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int n = i * kSortThreads + threadIdx.x;
      if (n < N) e[i] = sorted[n];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int n = i * kSortThreads + threadIdx.x;
    if (n < N) to[n] = e[i];
  }
}

// ---------------------------------------------------------------- sums
// Part u of the merged list: items [u * items, (u + 1) * items).  Partial sums [parts][D] fp32.
struct SumPlan {
  int64_t items, parts;
};

// Tokens among the first d items: the most t with key[t - 1] <= d - t.  A warp looks at 32 places at a time.
__device__ __forceinline__ int64_t merge_split(const uint2* sorted, int64_t N, int64_t rows, int64_t d) {
  const int lane = threadIdx.x % 32;
  int64_t lo = d > rows ? d - rows : 0, hi = d < N ? d : N;
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32, t = min(lo + (lane + 1) * step, hi);
    const unsigned yes = __ballot_sync(0xffffffffu, (int64_t)sorted[t - 1].x <= d - t);
    const int k = __popc(yes);  // the first k places
    if (k == 32) {
      lo = hi;
    } else {
      hi = min(lo + (k + 1) * step, hi) - 1;
      lo = lo + k * step;
    }
  }
  return lo;
}

// V consecutive elements of a lane (VEC false: 8 elements 32 apart), as they are fetched and as sums
template <typename T, bool VEC> struct Cols {
  static constexpr int N = VEC ? Vec<T>::N : 8;
  static constexpr int kWarp = 32 * N;  // columns of a warp
  struct Raw { uint4 w[VEC ? 1 : sizeof(T) / 2]; };
};
template <typename T, bool VEC>
__device__ __forceinline__ typename Cols<T, VEC>::Raw col_load(const T* row, int c0, int lane, int D, bool in) {
  typename Cols<T, VEC>::Raw f;
  if constexpr (VEC) {
    const int c = c0 + lane * Vec<T>::N;
    f.w[0] = ldg16_pred(row + (c < D ? c : 0), in && c < D);
  } else {
    T* e = reinterpret_cast<T*>(f.w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + i * 32 + lane;
      e[i] = in && c < D ? row[c] : from_f<T>(0.f);
    }
  }
  return f;
}
template <typename T, bool VEC>
__device__ __forceinline__ void col_add(float* acc, const typename Cols<T, VEC>::Raw& f) {
  if constexpr (VEC) {
    float x[Vec<T>::N];
    unpack16<T>(f.w[0], x);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) acc[i] += x[i];
  } else {
    const T* e = reinterpret_cast<const T*>(f.w);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += to_f(e[i]);
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

constexpr int kSumWarps = 4, kRowsAhead = 8;

// A warp's part: its tokens' rows are fetched kRowsAhead at a time, whatever rows of the table they belong to; a
// token of a later row first ends the rows before it.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kSumWarps * 32) embedding_sum_kernel(const uint2* sorted, const T* dy, int64_t dy_st,
                                                                       T* dtable, int64_t d_st, int64_t N,
                                                                       int64_t rows, int D, float scale, SumPlan p,
                                                                       int* heads, int* tails, float* head_sums,
                                                                       float* tail_sums) {
  using C = Cols<T, VEC>;
  const int lane = threadIdx.x % 32, c0 = blockIdx.y * C::kWarp;
  const int64_t u = (int64_t)blockIdx.x * kSumWarps + threadIdx.x / 32;
  let_next_start();
  if (u >= p.parts) return;
  wait_for_previous();
  const int64_t d0 = u * p.items, d1 = min(d0 + p.items, rows + N);
  int64_t t = merge_split(sorted, N, rows, d0);
  const int64_t t_end = merge_split(sorted, N, rows, d1), r_end = d1 - t_end;
  int64_t r = d0 - t;
  // the first row began in an earlier part
  bool begun = t > 0 && r < rows && (int64_t)sorted[t - 1].x == r;
  int head = -1;
  float acc[C::N];
#pragma unroll
  for (int i = 0; i < C::N; ++i) acc[i] = 0.f;
  auto end_row = [&] {
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
    begun = false;
    ++r;
  };
  bool any = false;  // the current row has tokens here
  for (int64_t w = t; w < t_end; w += 32) {
    const uint2 e = w + lane < t_end ? sorted[w + lane] : make_uint2((unsigned)rows, 0);
    const int n = (int)min((int64_t)32, t_end - w);
    for (int j = 0; j < n; j += kRowsAhead) {
      typename C::Raw f[kRowsAhead];
#pragma unroll
      for (int a = 0; a < kRowsAhead; ++a) {
        const unsigned token = __shfl_sync(0xffffffffu, e.y, (j + a) & 31);
        const bool in = j + a < n && __shfl_sync(0xffffffffu, e.x, (j + a) & 31) < (unsigned)rows;
        f[a] = col_load<T, VEC>(dy + (int64_t)token * dy_st, c0, lane, D, in);
      }
#pragma unroll
      for (int a = 0; a < kRowsAhead; ++a) {
        const int64_t key = __shfl_sync(0xffffffffu, e.x, (j + a) & 31);
        if (j + a >= n || key >= rows) break;
        while (r < key) {
          end_row();
          any = false;
        }
        col_add<T, VEC>(acc, f[a]);
        any = true;
      }
    }
  }
  while (r < r_end) {
    end_row();
    any = false;
  }
  int tail = -1;
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
// beginning are added in order, then its own.  A warp for a part; where a row took more than kManyParts, the CTA's
// eight warps take every eighth, and their sums are added in order.
constexpr int kManyParts = 16;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) embedding_cut_kernel(T* dtable, int64_t d_st, int D, float scale, int64_t parts,
                                                            const int* heads, const int* tails, float* head_sums,
                                                            float* tail_sums) {
  using C = Cols<T, VEC>;
  __shared__ float s[8][32][C::N + 1];
  __shared__ int64_t many[8];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, c0 = blockIdx.y * C::kWarp;
  const int64_t u = (int64_t)blockIdx.x * 8 + warp;
  wait_for_previous();
  const int head = u < parts ? heads[u] : -1;
  int64_t first = u;  // the part in which the row began
  if (head >= 0) {
    for (int64_t f0 = u - 1;; f0 -= 32) {
      const int64_t f = f0 - lane;
      const unsigned m = __ballot_sync(0xffffffffu, f < 0 || tails[f] >= -1);
      if (m != 0) {
        first = f0 - (__ffs(m) - 1);
        break;
      }
    }
  }
  const bool long_row = u - first > kManyParts;
  if (lane == 0) many[warp] = long_row ? first : -1;
  float acc[C::N];
  if (head >= 0 && !long_row) {
#pragma unroll
    for (int i = 0; i < C::N; ++i) acc[i] = 0.f;
#pragma unroll 4
    for (int64_t f = first; f <= u; ++f) {
      const float* q = part_at<C::N>(f == u ? head_sums : tail_sums, f, lane);
#pragma unroll
      for (int i = 0; i < C::N; ++i) acc[i] += q[i];
    }
#pragma unroll
    for (int i = 0; i < C::N; ++i) acc[i] *= scale;
    col_store<T, VEC>(dtable + head * d_st, c0, lane, D, acc);
  }
  __syncthreads();
  for (int k = 0; k < 8; ++k) {
    const int64_t from = many[k], to = (int64_t)blockIdx.x * 8 + k;
    if (from < 0) continue;
#pragma unroll
    for (int i = 0; i < C::N; ++i) acc[i] = 0.f;
#pragma unroll 8
    for (int64_t f = from + warp; f < to; f += 8) {
      const float* q = part_at<C::N>(tail_sums, f, lane);
#pragma unroll
      for (int i = 0; i < C::N; ++i) acc[i] += q[i];
    }
    __syncthreads();  // the sums of the row before this one are read
#pragma unroll
    for (int i = 0; i < C::N; ++i) s[warp][lane][i] = acc[i];
    __syncthreads();
    if (warp != k) continue;
#pragma unroll
    for (int i = 0; i < C::N; ++i) {
      float sum = 0.f;
      for (int w = 0; w < 8; ++w) sum += s[w][lane][i];
      acc[i] = scale * (sum + part_at<C::N>(head_sums, to, lane)[i]);
    }
    col_store<T, VEC>(dtable + head * d_st, c0, lane, D, acc);
  }
}

// ---------------------------------------------------------------- plans
static SortPlan sort_plan(int64_t N, int64_t rows) {
  SortPlan p;
  int bits = 1;
  while ((int64_t(1) << bits) <= rows) ++bits;  // the keys are 0 .. rows
  p.passes = (bits + 8) / 9;
  p.bits = (bits + p.passes - 1) / p.passes;
  const int64_t least = (N + kMostTiles - 1) / kMostTiles;
  p.tile = least <= kSortThreads ? kSortThreads : (least + kSortThreads - 1) / kSortThreads * kSortThreads;
  p.tiles = (int)((N + p.tile - 1) / p.tile);
  return p;
}
// Parts for two waves of warps over the column blocks; at least 8 items, so that a part's search and partial sums
// stay small beside its rows.
static SumPlan sum_plan(int64_t N, int64_t rows, int64_t D) {
  const int64_t total = N + rows, cols = (D + 255) / 256, parts = 148 * 64 / cols > 148 ? 148 * 64 / cols : 148;
  int64_t items = (total + parts - 1) / parts;
  if (items < 8) items = 8;
  return {items, (total + items - 1) / items};
}
static int64_t padded_cols(int64_t D) { return (D + 255) / 256 * 256; }

static size_t up(size_t n) { return (n + 255) / 256 * 256; }
struct Ws { size_t counts, a, b, heads, tails, head_sums, tail_sums, end; };
static Ws layout(int64_t N, int64_t rows, int64_t D) {
  const SortPlan sp = sort_plan(N, rows);
  const SumPlan su = sum_plan(N, rows, D);
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
  int lanes = 1;
  while (lanes < nv && lanes < 32) lanes *= 2;
  const int64_t rows_per_block = 256 / lanes * (nv <= lanes ? kLoads : 1), blocks = (N + rows_per_block - 1) / rows_per_block;
  auto go = [&](auto kernel) {
    kernel<<<(unsigned)blocks, 256, 0, s>>>(ids, static_cast<const T*>(table), table_st, static_cast<T*>(y), y_st, N, rows, nv,
                                            lanes, scale);
  };
  if (vec) nv <= lanes ? go(embedding_kernel<T, I, V, true>) : go(embedding_kernel<T, I, V, false>);
  else nv <= lanes ? go(embedding_kernel<T, I, 1, true>) : go(embedding_kernel<T, I, 1, false>);
  return launch_status("embedding_kernel");
}

template <typename T, bool VEC>
static int sums(const uint2* sorted, const void* dy, int64_t dy_st, void* dtable, int64_t d_st, int64_t N, int64_t rows,
                int64_t D, float scale, char* w, const Ws& at, cudaStream_t s) {
  const SumPlan p = sum_plan(N, rows, D);
  const unsigned cols = (unsigned)((D + Cols<T, VEC>::kWarp - 1) / Cols<T, VEC>::kWarp);
  int *heads = reinterpret_cast<int*>(w + at.heads), *tails = reinterpret_cast<int*>(w + at.tails);
  float *hs = reinterpret_cast<float*>(w + at.head_sums), *ts = reinterpret_cast<float*>(w + at.tail_sums);
  launch_dependent(embedding_sum_kernel<T, VEC>, dim3((unsigned)((p.parts + kSumWarps - 1) / kSumWarps), cols), kSumWarps * 32, 0,
                   s, sorted, static_cast<const T*>(dy), dy_st, static_cast<T*>(dtable), d_st, N, rows, (int)D, scale, p, heads,
                   tails, hs, ts);
  if (int e = launch_status("embedding_sum_kernel")) return e;
  launch_dependent(embedding_cut_kernel<T, VEC>, dim3((unsigned)((p.parts + 7) / 8), cols), 256, 0, s, static_cast<T*>(dtable),
                   d_st, (int)D, scale, p.parts, static_cast<const int*>(heads), static_cast<const int*>(tails), hs, ts);
  return launch_status("embedding_cut_kernel");
}

template <typename T, typename I>
static int gradient(const void* ids, const void* dy, int64_t dy_st, void* dtable, int64_t d_st, int64_t N, int64_t rows,
                    int64_t D, float scale, int64_t skip, char* w, cudaStream_t s) {
  const SortPlan p = sort_plan(N, rows);
  const Ws at = layout(N, rows, D);
  auto counts = reinterpret_cast<unsigned*>(w + at.counts);
  uint2* buf[2] = {reinterpret_cast<uint2*>(w + at.a), reinterpret_cast<uint2*>(w + at.b)};
  const bool one = N <= kOneTile;
  if (one && N > 0) {
    static std::atomic<uint64_t> ready{0};  // devices whose limit of shared memory is set
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
      cudaFuncSetAttribute(embedding_sort_one_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, kOneTile * 8);
      ready.fetch_or(bit, std::memory_order_relaxed);
    }
    embedding_sort_one_kernel<I><<<1, kSortThreads, kOneTile * 8, s>>>(ids, buf[0], (int)N, rows, skip, p);
    if (int e = launch_status("embedding_sort_one_kernel")) return e;
  } else if (N > 0) {
    embedding_count_kernel<I><<<p.tiles, kSortThreads, 0, s>>>(ids, N, rows, skip, p, counts);
    if (int e = launch_status("embedding_count_kernel")) return e;
    for (int k = 0; k < p.passes; ++k) {
      launch_dependent(embedding_sort_kernel<I>, dim3(p.tiles), kSortThreads, 0, s, ids, static_cast<const uint2*>(buf[(k + 1) % 2]),
                       buf[k % 2], N, rows, skip, p, k, counts);
      if (int e = launch_status("embedding_sort_kernel")) return e;
    }
  }
  const uint2* sorted = one ? buf[0] : buf[(p.passes + 1) % 2];
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
