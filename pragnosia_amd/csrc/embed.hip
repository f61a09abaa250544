// The token table's two directions: y_i = scale W[id_i], and dW[v] = scale sum over the tokens i with id_i = v of g_i.
//
// Both are bound by memory: the lookup moves n rows in and out, the gradient reads n rows and writes V. The gradient
// sorts the tokens by id (a stable counting sort: a row's terms are added in one order, with no atomics on values) in
// one launch, sums in a second and joins long runs in a third:
//
//   sort  Every workgroup owns a range of ids. It reads all n ids (they stay in the L2), counts those below its range
//         -- where its tokens start in the order -- and lists its own, ranked by id and position; then places them. No
//         workgroup waits for another.
//   sum   An id with at most kShort tokens (most of a vocabulary, zeros where there is none) is summed by one thread a
//         column vector, all its rows loaded at once. A longer run is summed in blocks of kBlock places of the order,
//         four waves a block, its rows shared among them; what is left of a run that goes on in another block is a
//         partial row.
//   join  A run's partial rows are added in order.
//
// A few tokens (kDirect) are one launch: a wave looks its ids up among all the tokens itself.
//
// Measured, fp32, 768 wide, word frequencies falling with the rank: 8192 tokens of 8192 words: lookup 8.3 us (50 MB: 6
// TB/s, part of it from the cache), sort 9, sum 10.5 (50 MB), join 3.5; 65536 of 32768: 56, 29, 89 (301 MB: 3.4 TB/s,
// short runs' rows and stores mixed), 6.
#include <algorithm>

#include "../include/pragnosia_lm.h"
#include "common.h"

namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kList = 768;     // tokens of a sorting wave that fit its LDS
constexpr int kAhead = 16;     // ids a lane of it loads at once
constexpr int kFew = 2;        // ids among 64 tokens that it tells apart one by one
constexpr int kIdBits = 9, kMaxRange = 1 << kIdBits;  // ids of a sorting workgroup, at most
constexpr int kDirect = 256;   // tokens up to which a gradient is one launch (256 of 8192 x 768: 8 us; three take 17)
constexpr int kShort = 8;    // tokens of an id summed by one thread
constexpr int kBlock = 64;   // places of the order summed by one workgroup: a lane each

template <class T>
struct Vec {};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  typedef f32x4 raw;
};
template <>
struct Vec<__bf16> {
  static constexpr int N = 8;
  typedef bf16x8 raw;
};

// y = scale W[id], kRows vectors of 16 bytes of W a thread, a launch's width apart: their ids, then their rows in
// flight together. kept: the ids in 32 bits, -1 outside the table, or null.
constexpr int kRows = 4;

template <class T, class O>
__global__ __launch_bounds__(256) void embed_rows(const int64_t* __restrict__ ids, const T* __restrict__ W, float scale,
                                                  O* __restrict__ y, int32_t* __restrict__ kept, int64_t n, int64_t V,
                                                  int d) {
  constexpr int N = Vec<T>::N;
  typedef O out_t __attribute__((__vector_size__(N * sizeof(O))));
  const int per = d / N;
  const int64_t total = n * per, width = (int64_t)gridDim.x * 256;
  for (int64_t e0 = (int64_t)blockIdx.x * 256 + threadIdx.x; e0 < total; e0 += width * kRows) {
    int64_t row[kRows], id[kRows];
    int c[kRows];
    typename Vec<T>::raw w[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int64_t e = min(e0 + u * width, total - 1);
      row[u] = e / per;
      c[u] = (int)(e - row[u] * per) * N;
      id[u] = ids[row[u]];
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const bool in = id[u] >= 0 && id[u] < V;
      if (!in) id[u] = -1;
      w[u] = *reinterpret_cast<const typename Vec<T>::raw*>(W + (in ? id[u] : 0) * d + c[u]);
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (e0 + u * width >= total) continue;
      if (kept != nullptr && c[u] == 0) kept[row[u]] = (int32_t)id[u];
      out_t o;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = id[u] >= 0 ? (O)(scale * (float)w[u][i]) : (O)0.f;
      *reinterpret_cast<out_t*>(y + row[u] * d + c[u]) = o;
    }
  }
}

// An id in 32 bits, -1 outside the table.
PGN_DEVICE int table_id(int64_t id, int64_t V) { return id >= 0 && id < V ? (int)id : -1; }

// Ids [blockIdx.x * range, ..): start[v] = the place of id v's first token in the order (start[V]: the number of
// tokens with an id), order[place] = position, sorted[place] = id. A wave reads a contiguous share of the ids in order,
// lists its tokens of the range and counts them by id, so a token's place is its id's start, the counts of the waves
// before, and its rank in its wave. A wave's list is kList tokens of LDS; a workgroup with more in some wave reads the
// ids again and lists them in `far` (n entries of scratch), where all of its waves know their places by then.
//
// Bound by the sixteen waves of each compute unit that look at every id between them: 65536 ids 29 us; counted first
// and listed in a second pass 38, with a branch around each load 53.
struct Token {
  int position;
  unsigned rank_id;  // rank among the wave's tokens of the id, and the id from the range's start in kIdBits
};

template <class I>
__global__ __launch_bounds__(kSortThreads) void embed_sort(const I* __restrict__ ids, int32_t* __restrict__ order,
                                                           int32_t* __restrict__ sorted, int32_t* __restrict__ start,
                                                           Token* __restrict__ far, int n, int V, int range) {
  extern __shared__ __align__(16) unsigned char smem[];
  // wave w's tokens of id r at [w * range + r]; then the place of the first of them
  int32_t* const count = reinterpret_cast<int32_t*>(smem + sizeof(Token) * kList * kSortWaves);
  __shared__ int32_t waves[2][kSortWaves];
  __shared__ int32_t first[kMaxRange];
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int v0 = blockIdx.x * range, v1 = min(V, v0 + range);
  const int share = ((n + kSortWaves - 1) / kSortWaves + 63) / 64 * 64, a = min(n, w * share), b = min(n, a + share);
  Token* list = reinterpret_cast<Token*>(smem) + w * kList;
  volatile int32_t* const own = count + w * range;  // (a wave's LDS operations are in order)
  const int bits = 32 - __clz(range - 1);
  int below = 0, mine = 0;  // a lane's ids below the range; the wave's tokens
  const unsigned long long lower = (1ull << l) - 1;
  auto append = [&](int i0, int x, int room) {
    const bool in = (unsigned)(x - v0) < (unsigned)(v1 - v0);
    const unsigned long long m = __ballot(in);
    if (m == 0) return;
    // the lanes with this lane's id: of the first kFew ids one by one (a few hot words), of what is left bit by bit
    // (65536 tokens of 64 ids of one range: 215 us, all one by one 460; with one hot word 33, all bit by bit 43)
    unsigned long long same = 0, left = m;
    for (int k = 0; k < kFew && left; ++k) {
      const int id = __builtin_amdgcn_readlane(x, __ffsll((long long)left) - 1);
      const unsigned long long lanes = __ballot(x == id);
      if (x == id) same = lanes;
      left &= ~lanes;
    }
    if (left) {
      unsigned long long rest = left;
      for (int k = 0; k < bits; ++k) {
        const bool one = (x - v0) >> k & 1;
        const unsigned long long ones = __ballot(one);
        rest &= one ? ones : ~ones;
      }
      if (left >> l & 1) same = rest;
    }
    if (in) {
      const int before = own[x - v0], rank = before + __popcll(same & lower), to = mine + __popcll(m & lower);
      if ((same & lower) == 0) own[x - v0] = before + __popcll(same);
      if (to < room) list[to] = {i0 + l, (unsigned)rank << kIdBits | (unsigned)(x - v0)};
    }
    mine += __popcll(m);
  };
  // kAhead ids a lane, -1 past the share or outside the table, the next ones under way; no load is behind a branch, or
  // each would be waited for by itself
  auto pass = [&](int room) {
    I next[kAhead];
    auto load = [&](int i0) {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) next[q] = ids[min(i0 + 64 * q + l, n - 1)];
    };
    for (int r = l; r < range; r += 64) own[r] = 0;
    below = mine = 0;
    load(a);
    for (int i0 = a; i0 < b; i0 += 64 * kAhead) {
      int x[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) x[q] = i0 + 64 * q + l < b ? table_id(next[q], V) : -1;
      if (i0 + 64 * kAhead < b) load(i0 + 64 * kAhead);
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        if (i0 + 64 * q >= b) break;
        below += (unsigned)x[q] < (unsigned)v0;
        append(i0 + 64 * q, x[q], room);
      }
    }
  };
  pass(kList);
  for (int o = 1; o < 64; o *= 2) below += __shfl_xor(below, o);
  if (l == 0) waves[0][w] = below, waves[1][w] = mine;
  __syncthreads();
  int base = 0, at = 0;
  bool fits = true;
  for (int q = 0; q < kSortWaves; ++q) {
    base += waves[0][q];
    if (q < w) at += waves[1][q];
    fits = fits && waves[1][q] <= kList;
  }
  if (!fits) {
    list = far + base + at;
    pass(n);
  }
  __syncthreads();
  // an id's tokens by wave: the counts of the waves before; and in all
  if (tid < range) {
    int s = 0;
    for (int q = 0; q < kSortWaves; ++q) {
      const int c = count[q * range + tid];
      count[q * range + tid] = s;
      s += c;
    }
    first[tid] = s;
  }
  __syncthreads();
  // an exclusive sum over the ids, by the first wave
  if (w == 0) {
    int run = base;
    for (int r0 = 0; r0 < range; r0 += 64) {
      const int c = r0 + l < range ? first[r0 + l] : 0;
      int s = c;
      for (int o = 1; o < 64; o *= 2) {
        const int t = __shfl_up(s, o);
        if (l >= o) s += t;
      }
      if (r0 + l < range) first[r0 + l] = run + s - c;
      if (v0 + r0 + l < v1) start[v0 + r0 + l] = run + s - c;
      run += __shfl(s, 63);
    }
    if (l == 0 && v1 == V) start[V] = run;
  }
  __syncthreads();
  for (int i = l; i < mine; i += 64) {
    const Token e = list[i];
    const int id = e.rank_id & (kMaxRange - 1), to = first[id] + own[id] + (int)(e.rank_id >> kIdBits);
    order[to] = e.position;
    sorted[to] = v0 + id;
  }
}

// s += the gradient rows of places [a, b), columns c .., U loaded at a time.
template <int U, class G>
PGN_DEVICE void sum_rows(const G* __restrict__ g, const int32_t* __restrict__ order, int a, int b, int64_t d, int c,
                         float (&s)[Vec<G>::N]) {
  constexpr int N = Vec<G>::N;
  for (int k = a; k < b; k += U) {
    typename Vec<G>::raw x[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = order[min(k + u, b - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < b) x[u] = *reinterpret_cast<const typename Vec<G>::raw*>(g + (int64_t)at[u] * d + c);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < b)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += (float)x[u][i];
  }
}

template <class G, class T>
PGN_DEVICE void put_row(T* p, const float (&s)[Vec<G>::N], float scale) {
  constexpr int N = Vec<G>::N;
  typedef T out_t __attribute__((__vector_size__(N * sizeof(T))));
  out_t o;
#pragma unroll
  for (int u = 0; u < N; ++u) o[u] = (T)(scale * s[u]);
  *reinterpret_cast<out_t*>(p) = o;
}

// The sums of four waves in order, in the first one's s. lds: 4 x 64 x N.
template <int N>
PGN_DEVICE void add_waves(float* lds, float (&s)[N], int w, int l) {
  __syncthreads();
#pragma unroll
  for (int u = 0; u < N; ++u) lds[(w * N + u) * 64 + l] = s[u];
  __syncthreads();
  if (w == 0)
    for (int q = 1; q < 4; ++q)
#pragma unroll
      for (int u = 0; u < N; ++u) s[u] += lds[(q * N + u) * 64 + l];
}

// Workgroups [0, blocks * chunks): places [kBlock q, kBlock q + kBlock) and a chunk of 64 column vectors, runs of more
// than kShort; a run that began in an earlier block leaves its partial row at 2 q, one that goes on in the next at
// 2 q + 1. The others: short runs, a thread an id and column vector.
template <class G, class T>
__global__ __launch_bounds__(256) void embed_sum(const G* __restrict__ g, const int32_t* __restrict__ order,
                                                 const int32_t* __restrict__ sorted, const int32_t* __restrict__ start,
                                                 float scale, T* __restrict__ dW, float* __restrict__ part, int V,
                                                 int d, int blocks, int chunks) {
  constexpr int N = Vec<G>::N;
  __shared__ float lds[4 * 64 * N];
  const int per = d / N;
  if ((int)blockIdx.x < blocks * chunks) {
    const int q = blockIdx.x / chunks, l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int col = (blockIdx.x - q * chunks) * 64 + l, c = min(col, per - 1) * N;
    const int lo = q * kBlock, hi = min(lo + kBlock, start[V]);
    // lane l: place lo + l, and its run
    const int v = lo + l < hi ? sorted[lo + l] : -1;
    const int from = v >= 0 ? start[v] : 0, to = v >= 0 ? start[v + 1] : 0;
    unsigned long long runs = __ballot(to - from > kShort && max(from, lo) == lo + l);
    while (runs) {
      const int lead = __ffsll((long long)runs) - 1;
      runs &= runs - 1;
      const int id = __shfl(v, lead), ra = __shfl(from, lead), rb = __shfl(to, lead), a = max(ra, lo), b = min(rb, hi);
      // a wave's share of the rows
      const int each = (b - a + 3) / 4, wa = min(b, a + w * each), wb = min(b, wa + each);
      float s[N] = {};
      sum_rows<8, G>(g, order, wa, wb, d, c, s);
      add_waves<N>(lds, s, w, l);
      if (w == 0 && col < per) {
        if (ra >= lo && rb <= hi) {
          put_row<G>(dW + (int64_t)id * d + c, s, scale);
        } else {
          float* p = part + (int64_t)(2 * q + (ra >= lo)) * d + c;
#pragma unroll
          for (int u = 0; u < N; ++u) p[u] = s[u];
        }
      }
    }
    return;
  }
  const int64_t total = (int64_t)V * per, stride = (int64_t)(gridDim.x - blocks * chunks) * 256;
  for (int64_t e = (int64_t)(blockIdx.x - blocks * chunks) * 256 + threadIdx.x; e < total; e += stride) {
    const int64_t v = e / per;
    const int c = (int)(e - v * per) * N, a = start[v], b = start[v + 1];
    if (b - a > kShort) continue;
    float s[N] = {};
    if (b - a <= 2)
      sum_rows<2, G>(g, order, a, b, d, c, s);
    else
      sum_rows<kShort, G>(g, order, a, b, d, c, s);
    put_row<G>(dW + v * d + c, s, scale);
  }
}

// The run that begins in block q and goes on past it: its partial rows in order, four waves a chunk of columns.
template <class G, class T>
__global__ __launch_bounds__(256) void embed_join(const int32_t* __restrict__ sorted, const int32_t* __restrict__ start,
                                                  float scale, T* __restrict__ dW, const float* __restrict__ part,
                                                  int V, int d, int chunks) {
  constexpr int N = Vec<G>::N;
  __shared__ float lds[4 * 64 * N];
  const int q = blockIdx.x / chunks, l = threadIdx.x & 63, w = threadIdx.x >> 6, per = d / N;
  const int lo = q * kBlock, hi = lo + kBlock;
  if (hi >= start[V]) return;
  const int v = sorted[hi - 1], from = start[v], to = start[v + 1];
  if (to - from <= kShort || from < lo || to <= hi) return;
  const int col = (blockIdx.x - q * chunks) * 64 + l, c = min(col, per - 1) * N;
  // block q's row at 2 q + 1, those of the blocks after it at 2 k
  const int rows = (to - 1) / kBlock - q + 1, each = (rows + 3) / 4, a = min(rows, w * each), b = min(rows, a + each);
  float s[N] = {};
  constexpr int U = 8;  // rows loaded at once (an id of 65536 tokens, 768 wide: 4 40 us, 8 27)
  for (int k = a; k < b; k += U) {
    f32x4 x[U][N / 4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(k + u, b - 1);
      const float* p = part + (int64_t)(2 * (q + at) + (at == 0)) * d + c;
#pragma unroll
      for (int i = 0; i < N / 4; ++i) x[u][i] = *reinterpret_cast<const f32x4*>(p + 4 * i);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < b)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += x[u][i / 4][i % 4];
  }
  add_waves<N>(lds, s, w, l);
  if (w == 0 && col < per) put_row<G>(dW + (int64_t)v * d + c, s, scale);
}

// n <= kDirect tokens: a wave owns kOwn ids and 64 column vectors. A row's terms are added in the order of their
// positions.
constexpr int kOwn = 8;

template <class G, class T, class I>
__global__ __launch_bounds__(256) void embed_direct(const G* __restrict__ g, const I* __restrict__ ids, float scale,
                                                    T* __restrict__ dW, int n, int V, int d) {
  constexpr int N = Vec<G>::N, U = 8;
  __shared__ int32_t all[kDirect];
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), per = d / N;
  if (tid < kDirect) all[tid] = tid < n ? table_id(ids[tid], V) : -1;
  __syncthreads();
  const int v0 = (blockIdx.x * 4 + w) * kOwn, col = blockIdx.y * 64 + l, c = min(col, per - 1) * N;
  // which tokens are the wave's, a bit each
  unsigned long long mine[kDirect / 64];
  int x[kDirect / 64];
#pragma unroll
  for (int q = 0; q < kDirect / 64; ++q) {
    x[q] = all[64 * q + l];
    mine[q] = __ballot(x[q] >= v0 && x[q] < v0 + kOwn);
  }
  for (int r = 0; r < kOwn; ++r) {
    const int v = v0 + r;
    if (v >= V) return;
    float s[N] = {};
#pragma unroll
    for (int q = 0; q < kDirect / 64; ++q) {
      if (mine[q] == 0) continue;
      unsigned long long left = __ballot(x[q] == v);
      while (left) {
        int at[U];
        typename Vec<G>::raw y[U];
        int k = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          at[u] = left ? 64 * q + __ffsll((long long)left) - 1 : -1;
          k += left != 0;
          left &= left - 1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < k) y[u] = *reinterpret_cast<const typename Vec<G>::raw*>(g + (int64_t)at[u] * d + c);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < k)
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] += (float)y[u][i];
      }
    }
    if (col < per) put_row<G>(dW + (int64_t)v * d + c, s, scale);
  }
}

constexpr int64_t kMaxTokens = (int64_t)1 << 27;  // (a rank in a wave, at most a sixteenth, is 32 - kIdBits bits)
constexpr int64_t kMaxWords = (int64_t)1 << 28;

// Ids a sorting workgroup owns: at most 256 workgroups where the counters allow (32 KB at most), as each reads all ids;
// no fewer, so that many tokens of a small table are shared out (65536 of 512 positions: 18 us; 32 ids each, 33).
int64_t sort_range(int64_t V) { return std::min<int64_t>((V + 255) / 256, kMaxRange); }

bool embed_shape_ok(int64_t n, int64_t V, int64_t d) {
  return n >= 0 && n <= kMaxTokens && V > 0 && V <= kMaxWords && d > 0 && d % 8 == 0 && d <= 65536 &&
         (n / kBlock + 1) * (d / 256 + 1) < (int64_t)1 << 22;  // launches of fewer than 2^32 threads
}

bool aligned(const void* p) { return ((uintptr_t)p % 16) == 0; }

int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

int64_t up4(int64_t x) { return (x + 3) / 4 * 4; }

template <class T, class O>
int launch_rows(const int64_t* ids, const void* W, float scale, void* y, int32_t* kept, int64_t n, int64_t V, int64_t d,
                hipStream_t st) {
  const int64_t blocks = (n * (d / Vec<T>::N) + 256 * kRows - 1) / (256 * kRows);
  hipLaunchKernelGGL((embed_rows<T, O>), dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(256), 0, st, ids,
                     (const T*)W, scale, (O*)y, kept, n, V, (int)d);
  PGN_RETURN_LAUNCH();
}

template <class G, class T, class I>
int launch_grad(const void* g, const I* ids, float scale, void* dW, int32_t* ws, int64_t n, int64_t V, int64_t d,
                hipStream_t st) {
  const int64_t per = d / Vec<G>::N, chunks = (per + 63) / 64, blocks = blocks_of(n);
  if (n <= kDirect) {
    hipLaunchKernelGGL((embed_direct<G, T, I>), dim3((unsigned)((V + 4 * kOwn - 1) / (4 * kOwn)), (unsigned)chunks),
                       dim3(256), 0, st, (const G*)g, ids, scale, (T*)dW, (int)n, (int)V, (int)d);
    PGN_RETURN_LAUNCH();
  }
  Token* far = (Token*)ws;
  int32_t *order = ws + 2 * up4(n), *sorted = order + up4(n), *start = sorted + up4(n);
  float* part = (float*)(start + up4(V + 1));
  const int range = (int)sort_range(V);
  const auto sort = embed_sort<I>;
  const int lists = (int)sizeof(Token) * kList * kSortWaves, lds = lists + 4 * kSortWaves * range;
  const hipError_t e = pgn_lds_limit((const void*)sort, lists + 4 * kSortWaves * kMaxRange);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(sort, dim3((unsigned)((V + range - 1) / range)), dim3(kSortThreads), lds, st, ids, order, sorted,
                     start, far, (int)n, (int)V, range);
  const int64_t whole = std::min<int64_t>((V * per + 255) / 256, 1 << 20);
  hipLaunchKernelGGL((embed_sum<G, T>), dim3((unsigned)(blocks * chunks + whole)), dim3(256), 0, st, (const G*)g, order,
                     sorted, start, scale, (T*)dW, part, (int)V, (int)d, (int)blocks, (int)chunks);
  hipLaunchKernelGGL((embed_join<G, T>), dim3((unsigned)((blocks - 1) * chunks)), dim3(256), 0, st, sorted, start,
                     scale, (T*)dW, part, (int)V, (int)d, (int)chunks);
  PGN_RETURN_LAUNCH();
}

template <class I>
int launch_grad_types(const void* g, int g_bf16, const I* ids, float scale, void* dW, int w_bf16, int32_t* ws,
                      int64_t n, int64_t V, int64_t d, hipStream_t st) {
  if (g_bf16) return w_bf16 ? launch_grad<__bf16, __bf16>(g, ids, scale, dW, ws, n, V, d, st)
                            : launch_grad<__bf16, float>(g, ids, scale, dW, ws, n, V, d, st);
  return w_bf16 ? launch_grad<float, __bf16>(g, ids, scale, dW, ws, n, V, d, st)
                : launch_grad<float, float>(g, ids, scale, dW, ws, n, V, d, st);
}

}  // namespace

extern "C" int pragnosia_embed_fwd(const int64_t* ids, const void* W, int w_bf16, float scale, void* y, int y_bf16,
                                   int32_t* kept, int64_t n, int64_t V, int64_t d, void* stream) {
  PGN_CHECK_ARG(embed_shape_ok(n, V, d) && W && aligned(W));
  if (n == 0) return PRAGNOSIA_OK;
  PGN_CHECK_ARG(ids && y && aligned(y));
  hipStream_t st = (hipStream_t)stream;
  if (w_bf16) return y_bf16 ? launch_rows<__bf16, __bf16>(ids, W, scale, y, kept, n, V, d, st)
                            : launch_rows<__bf16, float>(ids, W, scale, y, kept, n, V, d, st);
  return y_bf16 ? launch_rows<float, __bf16>(ids, W, scale, y, kept, n, V, d, st)
                : launch_rows<float, float>(ids, W, scale, y, kept, n, V, d, st);
}

extern "C" int64_t pragnosia_embed_bwd_workspace_bytes(int64_t n, int64_t V, int64_t d) {
  if (!embed_shape_ok(n, V, d)) return -1;
  return n <= kDirect ? 0 : (4 * up4(n) + up4(V + 1) + 2 * blocks_of(n) * d) * 4;
}

extern "C" int pragnosia_embed_bwd(const void* g, int g_bf16, const void* ids, int ids_64, float scale, void* dW,
                                   int w_bf16, void* workspace, int64_t workspace_bytes, int64_t n, int64_t V,
                                   int64_t d, void* stream) {
  PGN_CHECK_ARG(embed_shape_ok(n, V, d) && dW && aligned(dW) && (n == 0 || (g && ids && aligned(g) && aligned(ids))));
  const int64_t need = pragnosia_embed_bwd_workspace_bytes(n, V, d);
  PGN_CHECK_ARG(workspace_bytes >= need && (need == 0 || (workspace && aligned(workspace))));
  hipStream_t st = (hipStream_t)stream;
  int32_t* ws = (int32_t*)workspace;
  return ids_64 ? launch_grad_types(g, g_bf16, (const int64_t*)ids, scale, dW, w_bf16, ws, n, V, d, st)
                : launch_grad_types(g, g_bf16, (const int32_t*)ids, scale, dW, w_bf16, ws, n, V, d, st);
}
