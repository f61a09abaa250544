// The token table's two directions: y_i = scale W[id_i], and dW[v] = scale sum over the tokens i with id_i = v of g_i.
//
// Both are bound by memory: the lookup moves n rows in and out, the gradient reads n rows and writes V. The gradient
// sorts the tokens by id (a stable counting sort: a row's terms are added in the order of their positions, so the sum
// has one order and no atomics) in one launch, sums in a second and joins long runs in a third:
//
//   sort  Every workgroup owns a range of ids. It reads all n ids (they stay in the L2), counts those below its range
//         -- where its tokens start in the order -- and lists its own tokens' positions in order of position; then
//         places them by id. No workgroup waits for another.
//   sum   Ids with at most kRun tokens are summed whole, one workgroup a few ids, zeros where there is no token. A longer
//         run (a frequent word) is summed in blocks of kRun places of the order by other workgroups, each into a partial
//         row of its own.
//   join  A long run's partial rows are added in order.
#include <algorithm>

#include "../../include/lm/pragnosia_lm.h"
#include "common.h"

namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kRun = 32;  // tokens summed by one workgroup

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

// y = scale W[id], one vector of 16 bytes of W a thread.
template <class T, class O>
__global__ __launch_bounds__(256) void embed_rows(const int64_t* __restrict__ ids, const T* __restrict__ W, float scale,
                                                  O* __restrict__ y, int64_t n, int64_t V, int d) {
  constexpr int N = Vec<T>::N;
  const int per = d / N;
  const int64_t total = n * per;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
    const int64_t i = e / per;
    const int c = (int)(e - i * per) * N;
    const int64_t id = ids[i];
    typename Vec<T>::raw w{};
    const bool in = id >= 0 && id < V;
    if (in) w = *reinterpret_cast<const typename Vec<T>::raw*>(W + id * d + c);
    typedef O out_t __attribute__((__vector_size__(N * sizeof(O))));
    out_t o;
#pragma unroll
    for (int u = 0; u < N; ++u) o[u] = in ? (O)(scale * (float)w[u]) : (O)0.f;
    *reinterpret_cast<out_t*>(y + i * d + c) = o;
  }
}

// Ids [blockIdx.x * range, ..): start[v] = the place of id v's first token in the order (start[V] the number of tokens
// with an id in the table), order[place] = position. list: n entries, the unplaced positions and their ids.
__global__ __launch_bounds__(kSortThreads) void embed_sort(const int64_t* __restrict__ ids, int32_t* __restrict__ order,
                                                           int32_t* __restrict__ start, int32_t* __restrict__ list,
                                                           int n, int64_t V, int range) {
  extern __shared__ int32_t count_lds[];  // range: an id's tokens, then its next place
  volatile int32_t* count = count_lds;    // (read and written by different lanes of a wave)
  __shared__ int32_t waves[2][kSortWaves];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const int64_t v0 = (int64_t)blockIdx.x * range, v1 = min(V, v0 + range);
  // a wave reads a contiguous share of the ids, in order
  const int share = ((n + kSortWaves - 1) / kSortWaves + 63) / 64 * 64, a = min(n, w * share), b = min(n, a + share);
  int below = 0, mine = 0;
  for (int i = a + l; i < b; i += 64) {
    const int64_t id = ids[i];
    below += id >= 0 && id < v0;
    mine += id >= v0 && id < v1;
  }
  for (int o = 1; o < 64; o *= 2) below += __shfl_xor(below, o), mine += __shfl_xor(mine, o);
  if (l == 0) waves[0][w] = below, waves[1][w] = mine;
  for (int r = tid; r < range; r += kSortThreads) count[r] = 0;
  __syncthreads();
  int base = 0, before = 0, all = 0;
  for (int q = 0; q < kSortWaves; ++q) {
    base += waves[0][q];
    if (q < w) before += waves[1][q];
    all += waves[1][q];
  }
  // the range's tokens in order of position: list[base ..), counted by id
  int at = base + before;
  for (int i0 = a; i0 < b; i0 += 64) {
    const int64_t id = i0 + l < b ? ids[i0 + l] : -1;
    const bool in = id >= v0 && id < v1;
    const unsigned long long m = __ballot(in);
    if (in) {
      list[at + __popcll(m & ((1ull << l) - 1))] = i0 + l;
      atomicAdd(&count_lds[(int)(id - v0)], 1);
    }
    at += __popcll(m);
  }
  __syncthreads();
  // places: an exclusive sum over the range's counts, by the first wave
  if (w == 0) {
    int run = base;
    for (int r0 = 0; r0 < range; r0 += 64) {
      const int c = r0 + l < range ? count[r0 + l] : 0;
      int s = c;
      for (int o = 1; o < 64; o *= 2) {
        const int t = __shfl_up(s, o);
        if (l >= o) s += t;
      }
      if (r0 + l < range) count[r0 + l] = run + s - c;
      if (v0 + r0 + l < v1) start[v0 + r0 + l] = run + s - c;
      run += __shfl(s, 63);
    }
    if (l == 0 && v1 == V) start[V] = run;
  }
  __syncthreads();
  // each id's tokens placed in order: a wave takes the ids of its residue
  for (int i0 = 0; i0 < all; i0 += 64) {
    const int i = i0 + l < all ? list[base + i0 + l] : -1;
    const int r = i >= 0 ? (int)(ids[i] - v0) : -1;
    bool todo = r >= 0 && r % kSortWaves == w;
    unsigned long long left = __ballot(todo);
    while (left) {
      const int lead = __ffsll((unsigned long long)left) - 1, rl = __shfl(r, lead);
      const unsigned long long same = __ballot(todo && r == rl);
      const int place = count[rl];
      if (todo && r == rl) {
        order[place + __popcll(same & ((1ull << l) - 1))] = i;
        todo = false;
      }
      if (l == lead) count[rl] = place + __popcll(same);
      left &= ~same;
    }
  }
}

// Sum of the gradient rows of places [a, b), columns c ..
template <class G>
PGN_DEVICE void sum_rows(const G* __restrict__ g, const int32_t* __restrict__ order, int a, int b, int64_t d, int c,
                         float (&s)[Vec<G>::N]) {
  constexpr int N = Vec<G>::N;
#pragma unroll
  for (int u = 0; u < N; ++u) s[u] = 0.f;
  for (int k = a; k < b; ++k) {
    const typename Vec<G>::raw x = *reinterpret_cast<const typename Vec<G>::raw*>(g + (int64_t)order[k] * d + c);
#pragma unroll
    for (int u = 0; u < N; ++u) s[u] += (float)x[u];
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

// Workgroups [0, blocks): the places [kRun q, kRun q + kRun) of long runs, each into a partial row (the run that began
// earlier: row 2 q; the one that begins here: 2 q + 1). The others: whole ids, `per` threads' columns of one id each.
template <class G, class T>
__global__ __launch_bounds__(256) void embed_sum(const G* __restrict__ g, const int64_t* __restrict__ ids,
                                                 const int32_t* __restrict__ order, const int32_t* __restrict__ start,
                                                 float scale, T* __restrict__ dW, float* __restrict__ part, int64_t V,
                                                 int d, int blocks) {
  constexpr int N = Vec<G>::N;
  const int per = d / N;
  float s[N];
  if ((int)blockIdx.x < blocks) {
    const int q = blockIdx.x, lo = q * kRun, hi = min(lo + kRun, start[V]);
    if (lo >= hi) return;
    for (int side = 0; side < 2; ++side) {
      const int64_t v = ids[order[side ? hi - 1 : lo]];
      const int a = start[v], b = start[v + 1];
      if (b - a <= kRun) continue;
      if ((a < lo) != (side == 0)) continue;  // side 0: the run that began before this block; 1: the one that begins here
      for (int c = threadIdx.x * N; c < d; c += 256 * N) {
        sum_rows<G>(g, order, max(a, lo), min(b, hi), d, c, s);
#pragma unroll
        for (int u = 0; u < N; ++u) part[(int64_t)(2 * q + side) * d + c + u] = s[u];
      }
    }
    return;
  }
  const int64_t total = V * per;
  for (int64_t e = (int64_t)(blockIdx.x - blocks) * 256 + threadIdx.x; e < total;
       e += (int64_t)(gridDim.x - blocks) * 256) {
    const int64_t v = e / per;
    const int c = (int)(e - v * per) * N, a = start[v], b = start[v + 1];
    if (b - a > kRun) continue;
    sum_rows<G>(g, order, a, b, d, c, s);
    put_row<G>(dW + v * d + c, s, scale);
  }
}

// The long run that begins in block q: its partial rows in order.
template <class G, class T>
__global__ __launch_bounds__(256) void embed_join(const int64_t* __restrict__ ids, const int32_t* __restrict__ order,
                                                  const int32_t* __restrict__ start, float scale, T* __restrict__ dW,
                                                  const float* __restrict__ part, int64_t V, int d) {
  constexpr int N = Vec<G>::N;
  const int q = blockIdx.x, lo = q * kRun, hi = min(lo + kRun, start[V]);
  if (lo >= hi) return;
  const int64_t v = ids[order[hi - 1]];
  const int a = start[v], b = start[v + 1];
  if (b - a <= kRun || a < lo) return;
  const int last = (b - 1) / kRun;
  for (int c = threadIdx.x * N; c < d; c += 256 * N) {
    float s[N];
#pragma unroll
    for (int u = 0; u < N; ++u) s[u] = part[(int64_t)(2 * q + 1) * d + c + u];
    for (int k = q + 1; k <= last; ++k)
#pragma unroll
      for (int u = 0; u < N; ++u) s[u] += part[(int64_t)(2 * k) * d + c + u];
    put_row<G>(dW + v * d + c, s, scale);
  }
}

constexpr int64_t kMaxTokens = (int64_t)1 << 28;  // launches of fewer than 2^32 threads

// Ids a sorting workgroup owns: about 512 workgroups, their counters at most 16 KB.
int64_t sort_range(int64_t V) { return std::min<int64_t>(std::max<int64_t>((V + 511) / 512, 32), 4096); }

bool embed_shape_ok(int64_t n, int64_t V, int64_t d) {
  return n >= 0 && n <= kMaxTokens && V > 0 && V <= kMaxTokens && d > 0 && d % 8 == 0 && d <= 65536;
}

bool aligned(const void* p) { return ((uintptr_t)p % 16) == 0; }

int64_t runs(int64_t n) { return (n + kRun - 1) / kRun; }

int64_t up4(int64_t x) { return (x + 3) / 4 * 4; }

template <class T, class O>
int launch_rows(const int64_t* ids, const void* W, float scale, void* y, int64_t n, int64_t V, int64_t d,
                hipStream_t st) {
  const int64_t blocks = (n * (d / Vec<T>::N) + 255) / 256;
  hipLaunchKernelGGL((embed_rows<T, O>), dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(256), 0, st, ids,
                     (const T*)W, scale, (O*)y, n, V, (int)d);
  PGN_RETURN_LAUNCH();
}

template <class G, class T>
int launch_grad(const void* g, const int64_t* ids, float scale, void* dW, int32_t* ws, int64_t n, int64_t V, int64_t d,
                hipStream_t st) {
  int32_t *order = ws, *list = ws + up4(n), *start = ws + 2 * up4(n);
  float* part = (float*)(start + up4(V + 1));
  const int range = (int)sort_range(V);
  hipLaunchKernelGGL(embed_sort, dim3((unsigned)((V + range - 1) / range)), dim3(kSortThreads), range * 4, st, ids,
                     order, start, list, (int)n, V, range);
  const int64_t blocks = runs(n), whole = std::min<int64_t>((V * (d / Vec<G>::N) + 255) / 256, 1 << 20);
  hipLaunchKernelGGL((embed_sum<G, T>), dim3((unsigned)(blocks + whole)), dim3(256), 0, st, (const G*)g, ids, order,
                     start, scale, (T*)dW, part, V, (int)d, (int)blocks);
  if (n > kRun)
    hipLaunchKernelGGL((embed_join<G, T>), dim3((unsigned)blocks), dim3(256), 0, st, ids, order, start, scale, (T*)dW,
                       part, V, (int)d);
  PGN_RETURN_LAUNCH();
}

}  // namespace

extern "C" int pragnosia_embed_fwd(const int64_t* ids, const void* W, int w_bf16, float scale, void* y, int y_bf16,
                                   int64_t n, int64_t V, int64_t d, void* stream) {
  PGN_CHECK_ARG(embed_shape_ok(n, V, d) && W && aligned(W));
  if (n == 0) return PRAGNOSIA_OK;
  PGN_CHECK_ARG(ids && y && aligned(y));
  hipStream_t st = (hipStream_t)stream;
  if (w_bf16) return y_bf16 ? launch_rows<__bf16, __bf16>(ids, W, scale, y, n, V, d, st)
                            : launch_rows<__bf16, float>(ids, W, scale, y, n, V, d, st);
  return y_bf16 ? launch_rows<float, __bf16>(ids, W, scale, y, n, V, d, st)
                : launch_rows<float, float>(ids, W, scale, y, n, V, d, st);
}

extern "C" int64_t pragnosia_embed_bwd_workspace_bytes(int64_t n, int64_t V, int64_t d) {
  if (!embed_shape_ok(n, V, d)) return -1;
  return (2 * up4(n) + up4(V + 1) + (n > kRun ? 2 * runs(n) * d : 0)) * 4;
}

extern "C" int pragnosia_embed_bwd(const void* g, int g_bf16, const int64_t* ids, float scale, void* dW, int w_bf16,
                                   void* workspace, int64_t workspace_bytes, int64_t n, int64_t V, int64_t d,
                                   void* stream) {
  PGN_CHECK_ARG(embed_shape_ok(n, V, d) && dW && aligned(dW) && (n == 0 || (g && ids && aligned(g))));
  PGN_CHECK_ARG(workspace && aligned(workspace) && workspace_bytes >= pragnosia_embed_bwd_workspace_bytes(n, V, d));
  hipStream_t st = (hipStream_t)stream;
  int32_t* ws = (int32_t*)workspace;
  if (g_bf16) return w_bf16 ? launch_grad<__bf16, __bf16>(g, ids, scale, dW, ws, n, V, d, st)
                            : launch_grad<__bf16, float>(g, ids, scale, dW, ws, n, V, d, st);
  return w_bf16 ? launch_grad<float, __bf16>(g, ids, scale, dW, ws, n, V, d, st)
                : launch_grad<float, float>(g, ids, scale, dW, ws, n, V, d, st);
}
