// Losses of a head l = h W^T over a vocabulary, and their gradients, with no logits kept: cross entropy of labels and
// distillation from a teacher's top logits (formulas at pragnosia_head_fwd).
//
// Forward: each tile of 256 words x 256 tokens is one matrix product whose logits stay in the accumulators; every wave
// reduces its 128 words per token to a maximum and a sum of exponentials (two, where the cross entropy and a softened
// distillation loss share the pass), in fp32. A last kernel joins a row's pieces. The operands are swapped (words are
// the product's rows), so a token's words lie in one lane's registers and the reduction is two lane exchanges a token.
//
// Backward: the logits are formed again per piece of the vocabulary, turned into dl in the accumulators and rounded to
// bf16 (relative 2^-8 of each element, the gradient of a logit, the operands' own precision) into a workspace of the
// piece's columns; dh += dl W and dW = dl^T h are products over it.
#include <algorithm>

#include "../../include/lm/pragnosia_lm.h"
#include "gemm_tile.h"

using namespace pgn;

namespace {

constexpr int kWaveWords = 128;  // words a wave reduces: one piece of a row's softmax

// The workspace of one piece's dl: at most this many bytes (but at least one column of tiles).
constexpr int64_t kPieceBytes = (int64_t)256 << 20;

struct Plan {
  int64_t n_pad, v_piece, pieces;
};

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

Plan plan(int64_t n, int64_t V) {
  Plan p;
  p.n_pad = round_up(n, kGemmTile);
  const int64_t v_pad = round_up(V, kGemmTile);
  const int64_t most = std::max<int64_t>(kGemmTile, kPieceBytes / (2 * p.n_pad) / kGemmTile * kGemmTile);
  p.pieces = (v_pad + most - 1) / most;
  p.v_piece = round_up((v_pad + p.pieces - 1) / p.pieces, kGemmTile);
  p.pieces = (v_pad + p.v_piece - 1) / p.v_piece;
  return p;
}

// Lane exchange of the groups of 16: the maximum, and the sum, over a column's four lane groups, in every one of them.
PGN_DEVICE float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
PGN_DEVICE float column_sum(float x) { return swap_add<32>(swap_add<16>(x, x), swap_add<16>(x, x)); }

// ---------------------------------------------------------------------------------------------------------------
// The teacher's distribution over its entries, a wave a row.
__global__ __launch_bounds__(256) void head_teacher(const int64_t* __restrict__ ids, const float* __restrict__ z,
                                                    float inv_tau, int32_t* __restrict__ entry,
                                                    float* __restrict__ p, float* __restrict__ psum,
                                                    float* __restrict__ ent, int64_t n, int64_t V, int64_t K) {
  const int l = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  ids += row * K, z += row * K, entry += row * K, p += row * K;
  float m = -INFINITY;
  for (int64_t k = l; k < K; k += 64)
    if (ids[k] >= 0 && ids[k] < V) m = fmaxf(m, z[k] * inv_tau);
  for (int o = 1; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
  const bool some = m > -INFINITY;
  float sum = 0.f;
  for (int64_t k = l; k < K; k += 64)
    if (some && ids[k] >= 0 && ids[k] < V) sum += expf(z[k] * inv_tau - m);
  for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
  const float inv = some ? 1.f / sum : 0.f, log_sum = some ? logf(sum) : 0.f;
  float e = 0.f;
  for (int64_t k = l; k < K; k += 64) {
    const bool on = some && ids[k] >= 0 && ids[k] < V;
    const float x = on ? z[k] * inv_tau - m : -INFINITY;
    const float pk = on ? expf(x) * inv : 0.f;
    entry[k] = on ? (int32_t)ids[k] : -1;
    p[k] = pk;
    if (pk > 0.f) e += pk * (x - log_sum);
  }
  for (int o = 1; o < 64; o *= 2) e += __shfl_xor(e, o);
  if (l == 0) {
    psum[row] = some ? 1.f : 0.f;
    ent[row] = e;
  }
}

// The student's logits of the teacher's entries, zl[i][k] = h_i . W_entry; a wave a row, 16 lanes an entry.
__global__ __launch_bounds__(256) void head_entry_logits(const __bf16* __restrict__ h, const __bf16* __restrict__ W,
                                                         const int32_t* __restrict__ entry, float* __restrict__ zl,
                                                         int64_t n, int64_t d, int64_t K) {
  const int l = threadIdx.x & 63, q = l >> 4, j = l & 15;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  const __bf16* hr = h + row * d;
  for (int64_t k0 = 0; k0 < K; k0 += 4) {
    const int64_t k = k0 + q;
    const int e = k < K ? entry[row * K + k] : -1;
    float s = 0.f;
    if (e >= 0) {
      const __bf16* wr = W + (int64_t)e * d;
      for (int64_t c = 8 * j; c < d; c += 128) {
        const bf16x8 a = *reinterpret_cast<const bf16x8*>(hr + c), b = *reinterpret_cast<const bf16x8*>(wr + c);
#pragma unroll
        for (int u = 0; u < 8; ++u) s += (float)a[u] * (float)b[u];
      }
    }
    s = group_sum<16>(s);
    if (j == 0 && k < K) zl[row * K + k] = s;
  }
}

struct FwdOut {
  float *m, *s0, *s1;  // pieces x n: maximum of l, sums of exp(scale0 (l - m)) and exp(scale1 (l - m))
  float* label;        // n: the label's logit (written only where the label is in range)
};

// One tile's logits reduced. NEXP sums of exponentials, of scale0 l and scale1 l.
template <int NEXP>
__global__ __launch_bounds__(kGemmThreads) void head_logits(Operand h, Operand W, const int64_t* __restrict__ y,
                                                            float scale0, float scale1, FwdOut out, int64_t d) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int64_t tx = (W.rows + kGemmTile - 1) / kGemmTile, ty = (h.rows + kGemmTile - 1) / kGemmTile;
  const int64_t item = xcd_item(blockIdx.x, tx * ty);
  if (item < 0) return;
  int64_t ix, iy;
  band_tile(item, tx, ty, ix, iy);
  f32x4 acc[8][4];
  gemm_tile<false, false>(W, h, ix * kGemmTile, iy * kGemmTile, 0, d, smem, acc);
  const WaveIdx t = wave_idx();
  const int64_t v0 = ix * kGemmTile + (t.w & 1) * kWaveWords, i0 = iy * kGemmTile + (t.w >> 1) * 64, n = h.rows;
  const float c0 = scale0 * kLog2e, c1 = scale1 * kLog2e;
  if (v0 + kWaveWords > W.rows) {
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (v0 + 16 * a + 4 * t.g + r >= W.rows)
#pragma unroll
          for (int b = 0; b < 4; ++b) acc[a][b][r] = -INFINITY;
  }
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int64_t row = i0 + 16 * b + t.i;
    if (y != nullptr) {
      const int64_t at = row < n ? y[row] - v0 : -1;
      if (__ballot(at >= 0 && at < kWaveWords)) {
        const int own = (at >= 0 && at < kWaveWords) ? (int)at - 4 * t.g : -1;
#pragma unroll
        for (int a = 0; a < 8; ++a)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (own == 16 * a + r && v0 + at < W.rows) out.label[row] = acc[a][b][r];
      }
    }
    float m = acc[0][b][0];
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[a][b][r]);
    m = column_max(m);
    const float base = m > -INFINITY ? m : 0.f;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s0 += exp2_hw((acc[a][b][r] - base) * c0);
        if constexpr (NEXP == 2) s1 += exp2_hw((acc[a][b][r] - base) * c1);
      }
    s0 = column_sum(s0);
    if constexpr (NEXP == 2) s1 = column_sum(s1);
    if (t.g == 0 && row < n) {
      const int64_t o = (v0 / kWaveWords) * n + row;
      out.m[o] = m;
      out.s0[o] = s0;
      if constexpr (NEXP == 2) out.s1[o] = s1;
    }
  }
}

// A row's pieces joined: a thread a row.
__global__ __launch_bounds__(64) void head_join(FwdOut in, int64_t pieces, float scale0, float scale1,
                                                const int64_t* __restrict__ y, float* __restrict__ ce,
                                                float* __restrict__ lse, const float* __restrict__ ent,
                                                const float* __restrict__ psum, const float* __restrict__ p,
                                                const float* __restrict__ zl, float tau, float* __restrict__ kd,
                                                float* __restrict__ lse_t, int second, int64_t n, int64_t V,
                                                int64_t K) {
  const int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (row >= n) return;
  float m = -INFINITY;
  for (int64_t q = 0; q < pieces; ++q) m = fmaxf(m, in.m[q * n + row]);
  float s0 = 0.f, s1 = 0.f;
  for (int64_t q = 0; q < pieces; ++q) {
    const float mq = in.m[q * n + row] - m;
    s0 += in.s0[q * n + row] * expf(mq * scale0);
    if (second) s1 += in.s1[q * n + row] * expf(mq * scale1);
  }
  const float l0 = m * scale0 + logf(s0), l1 = second ? m * scale1 + logf(s1) : l0;
  if (y != nullptr) {
    lse[row] = l0;
    ce[row] = y[row] >= 0 && y[row] < V ? l0 - in.label[row] : 0.f;
  }
  if (K > 0) {
    float dot = 0.f;
    for (int64_t k = 0; k < K; ++k) {
      const float pk = p[row * K + k];
      if (pk > 0.f) dot += pk * zl[row * K + k];
    }
    lse_t[row] = l1;
    kd[row] = psum[row] > 0.f ? tau * tau * (ent[row] - dot / tau + l1) : 0.f;
  }
}

// ---------------------------------------------------------------------------------------------------------------
struct BwdIn {
  const float *g_ce, *g_lse, *g_kd, *lse, *lse_t, *psum;
  const int64_t* y;
  float tau;
};

// dl of a piece of the vocabulary: words v_begin .. v_begin + ld of the workspace's rows (n_pad, ld). Word and token
// rows past the ends get zeros.
template <int NEXP>
__global__ __launch_bounds__(kGemmThreads) void head_dlogits(Operand h, Operand W, BwdIn in, float scale0,
                                                             float scale1, __bf16* __restrict__ dl, int64_t ld,
                                                             int64_t v_begin, int64_t d) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int64_t tx = ld / kGemmTile, ty = (h.rows + kGemmTile - 1) / kGemmTile;
  const int64_t item = xcd_item(blockIdx.x, tx * ty);
  if (item < 0) return;
  int64_t ix, iy;
  band_tile(item, tx, ty, ix, iy);
  f32x4 acc[8][4];
  gemm_tile<false, false>(W, h, v_begin + ix * kGemmTile, iy * kGemmTile, 0, d, smem, acc);
  const WaveIdx t = wave_idx();
  const int64_t c0 = ix * kGemmTile + (t.w & 1) * kWaveWords, v0 = v_begin + c0;
  const int64_t i0 = iy * kGemmTile + (t.w >> 1) * 64, n = h.rows;
  const float e0 = scale0 * kLog2e, e1 = scale1 * kLog2e;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int64_t row = i0 + 16 * b + t.i;
    const bool live = row < n;
    // weights of the two softmaxes in dl, and the label
    const int64_t label = live && in.y != nullptr ? in.y[row] : -1;
    const bool labelled = label >= 0 && label < W.rows;
    const float gc = live && labelled && in.g_ce != nullptr ? in.g_ce[row] : 0.f;
    const float w_ce = gc + (live && in.g_lse != nullptr ? in.g_lse[row] : 0.f);
    const float w_kd = live && in.g_kd != nullptr ? in.g_kd[row] * in.tau * in.psum[row] : 0.f;
    float w0, w1 = 0.f, l0, l1 = 0.f;
    if constexpr (NEXP == 2) {
      w0 = w_ce, w1 = w_kd;
      l0 = live ? in.lse[row] * kLog2e : 0.f, l1 = live ? in.lse_t[row] * kLog2e : 0.f;
    } else {
      w0 = w_ce + w_kd;
      l0 = live ? (in.lse != nullptr ? in.lse[row] : in.lse_t[row]) * kLog2e : 0.f;
    }
    const bool any = w_ce != 0.f || w_kd != 0.f || gc != 0.f;
    const int at = labelled && gc != 0.f && label >= v0 && label < v0 + kWaveWords ? (int)(label - v0) - 4 * t.g : -1;
    const bool hit = __ballot(at >= 0) != 0;
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = w0 * exp2_hw(acc[a][b][r] * e0 - l0);
        if constexpr (NEXP == 2) x[r] += w1 * exp2_hw(acc[a][b][r] * e1 - l1);
        if (hit && at == 16 * a + r) x[r] -= gc;
        if (!any || v0 + 16 * a + 4 * t.g + r >= W.rows) x[r] = 0.f;
      }
      *reinterpret_cast<bf16x4*>(dl + row * ld + c0 + 16 * a + 4 * t.g) = to_bf16x4(x);
    }
  }
}

// dl at the teacher's entries, whole: a thread an entry. Repeated ids write the same value.
__global__ __launch_bounds__(256) void head_entry_dl(BwdIn in, const int32_t* __restrict__ entry,
                                                     const float* __restrict__ p, const float* __restrict__ zl,
                                                     __bf16* __restrict__ dl, int64_t ld, int64_t v_begin, int64_t n,
                                                     int64_t V, int64_t K) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n * K) return;
  const int64_t row = e / K;
  const int v = entry[e];
  if (v < v_begin || v >= v_begin + ld) return;
  const int64_t label = in.y != nullptr ? in.y[row] : -1;
  const bool labelled = label >= 0 && label < V;
  const float gc = labelled && in.g_ce != nullptr ? in.g_ce[row] : 0.f;
  const float w_ce = gc + (in.g_lse != nullptr ? in.g_lse[row] : 0.f), gk = in.g_kd[row] * in.tau;
  float x = 0.f;
  if (w_ce != 0.f || gk != 0.f || gc != 0.f) {
    float pk = 0.f;
    for (int64_t k = 0; k < K; ++k)
      if (entry[row * K + k] == v) pk += p[row * K + k];
    const float l = zl[e];
    x = gk * (in.psum[row] * expf(l / in.tau - in.lse_t[row]) - pk);
    if (w_ce != 0.f) x += w_ce * expf(l - in.lse[row]);
    if (label == v) x -= gc;
  }
  dl[row * ld + (v - v_begin)] = (__bf16)x;
}

// dh (+)= dl W over a piece (the first workgroups) and dW = dl^T h of the piece (the others).
struct GradArgs {
  Operand dl_rows, dl_words;  // dl by its rows (n_pad), contracted over words / over tokens
  Operand W, h;               // W's rows of the piece; h
  int64_t n, d, words, n_pad, ld;
  __bf16* dh;
  float* dh_acc;   // fp32 sums where there are several pieces
  int first, last;
  void* dW;        // the piece's rows
  int dw_f32;
  int64_t items_h, items_w;
};

__global__ __launch_bounds__(kGemmThreads) void head_grads(GradArgs q) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int64_t tx = (q.d + kGemmTile - 1) / kGemmTile;
  f32x4 acc[8][4];
  int64_t item = xcd_item(blockIdx.x, q.items_h + q.items_w);
  if (item < 0) return;
  const WaveIdx t = wave_idx();
  int64_t ix, iy;
  if (item < q.items_h) {
    iy = item / tx, ix = item - iy * tx;
    gemm_tile<true, false>(q.W, q.dl_rows, ix * kGemmTile, iy * kGemmTile, 0, q.words, smem, acc);
    const int64_t c0 = ix * kGemmTile + (t.w & 1) * 128, i0 = iy * kGemmTile + (t.w >> 1) * 64;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int64_t row = i0 + 16 * b + t.i;
      if (row >= q.n) continue;
#pragma unroll
      for (int a = 0; a < 8; ++a) {
        const int64_t c = c0 + 16 * a + 4 * t.g;
        if (c >= q.d) continue;
        f32x4 x = acc[a][b];
        if (!q.first) x += *reinterpret_cast<const f32x4*>(q.dh_acc + row * q.d + c);
        if (q.last)
          *reinterpret_cast<bf16x4*>(q.dh + row * q.d + c) = to_bf16x4(x);
        else
          *reinterpret_cast<f32x4*>(q.dh_acc + row * q.d + c) = x;
      }
    }
  } else {
    item -= q.items_h;
    iy = item / tx, ix = item - iy * tx;
    gemm_tile<true, true>(q.h, q.dl_words, ix * kGemmTile, iy * kGemmTile, 0, q.n, smem, acc);
    const int64_t c0 = ix * kGemmTile + (t.w & 1) * 128, i0 = iy * kGemmTile + (t.w >> 1) * 64;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int64_t row = i0 + 16 * b + t.i;
      if (row >= q.words) continue;
#pragma unroll
      for (int a = 0; a < 8; ++a) {
        const int64_t c = c0 + 16 * a + 4 * t.g;
        if (c >= q.d) continue;
        if (q.dw_f32)
          *reinterpret_cast<f32x4*>((float*)q.dW + row * q.d + c) = acc[a][b];
        else
          *reinterpret_cast<bf16x4*>((__bf16*)q.dW + row * q.d + c) = to_bf16x4(acc[a][b]);
      }
    }
  }
}

bool head_shape_ok(int64_t n, int64_t V, int64_t d, int64_t K) {
  return n > 0 && n <= (int64_t)1 << 24 && V > 0 && V <= (int64_t)1 << 24 && d > 0 && d % 8 == 0 && d <= 65536 &&
         K >= 0 && K <= 65536 && round_up(n, kGemmTile) / kGemmTile * (round_up(V, kGemmTile) / kGemmTile) < 1 << 22 &&
         n * K < (int64_t)1 << 31;  // launches of fewer than 2^32 threads
}

bool aligned(const void* p) { return ((uintptr_t)p % 16) == 0; }

int64_t head_pieces(int64_t V) { return round_up(V, kGemmTile) / kWaveWords; }

}  // namespace

extern "C" int pragnosia_lm_abi_version(void) { return 1; }

extern "C" int64_t pragnosia_head_fwd_workspace_bytes(int64_t n, int64_t V, int64_t d, int64_t K) {
  if (!head_shape_ok(n, V, d, K)) return -1;
  return (3 * head_pieces(V) + 2) * n * (int64_t)sizeof(float);
}

extern "C" int pragnosia_head_fwd(const void* h, const void* W, const int64_t* y, const int64_t* ids, const float* z,
                                  float tau, float* ce, float* lse, float* kd, float* lse_t, float* psum,
                                  int32_t* entry, float* p, float* zl, void* workspace, int64_t workspace_bytes,
                                  int64_t n, int64_t V, int64_t d, int64_t K, void* stream) {
  PGN_CHECK_ARG(head_shape_ok(n, V, d, K));
  PGN_CHECK_ARG(h && W && (y || ids) && aligned(h) && aligned(W));
  PGN_CHECK_ARG(!y || (ce && lse));
  PGN_CHECK_ARG((ids != nullptr) == (K > 0) && (z != nullptr) == (K > 0));
  PGN_CHECK_ARG(K == 0 || (kd && lse_t && psum && entry && p && zl));
  PGN_CHECK_ARG(tau > 0.f && tau < INFINITY);
  PGN_CHECK_ARG(workspace && aligned(workspace) && workspace_bytes >= pragnosia_head_fwd_workspace_bytes(n, V, d, K));
  hipStream_t st = (hipStream_t)stream;
  const int64_t pieces = head_pieces(V);
  float* f = (float*)workspace;
  const FwdOut out{f, f + pieces * n, f + 2 * pieces * n, f + 3 * pieces * n};
  float* ent = f + (3 * pieces + 1) * n;
  const Operand ho{(const __bf16*)h, d, n}, Wo{(const __bf16*)W, d, V};
  hipError_t e = pgn_lds_limit((const void*)head_logits<1>, kGemmLds);
  if (e == hipSuccess) e = pgn_lds_limit((const void*)head_logits<2>, kGemmLds);
  if (e != hipSuccess) return (int)e;
  if (K > 0) {
    hipLaunchKernelGGL(head_teacher, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, ids, z, 1.f / tau, entry, p, psum,
                       ent, n, V, K);
    hipLaunchKernelGGL(head_entry_logits, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, ho.p, Wo.p, entry, zl, n, d,
                       K);
  }
  const int second = y && K > 0 && tau != 1.f;
  const float scale0 = y ? 1.f : 1.f / tau, scale1 = 1.f / tau;
  const int64_t items = round_up(V, kGemmTile) / kGemmTile * (round_up(n, kGemmTile) / kGemmTile);
  if (second)
    hipLaunchKernelGGL(head_logits<2>, dim3(xcd_grid(items)), dim3(kGemmThreads), kGemmLds, st, ho, Wo, y, scale0,
                       scale1, out, d);
  else
    hipLaunchKernelGGL(head_logits<1>, dim3(xcd_grid(items)), dim3(kGemmThreads), kGemmLds, st, ho, Wo, y, scale0,
                       scale1, out, d);
  hipLaunchKernelGGL(head_join, dim3((unsigned)((n + 63) / 64)), dim3(64), 0, st, out, pieces, scale0, scale1, y, ce,
                     lse, ent, psum, p, zl, tau, kd, lse_t, second, n, V, K);
  PGN_RETURN_LAUNCH();
}

extern "C" int64_t pragnosia_head_bwd_workspace_bytes(int64_t n, int64_t V, int64_t d) {
  if (!head_shape_ok(n, V, d, 0)) return -1;
  const Plan pl = plan(n, V);
  return pl.n_pad * pl.v_piece * 2 + (pl.pieces > 1 ? n * d * 4 : 0);
}

extern "C" int pragnosia_head_bwd(const float* g_ce, const float* g_lse, const float* g_kd, const void* h,
                                  const void* W, const int64_t* y, const float* lse, const float* lse_t,
                                  const float* psum, const int32_t* entry, const float* p, const float* zl, float tau,
                                  void* dh, void* dW, int dw_f32, void* workspace, int64_t workspace_bytes, int64_t n,
                                  int64_t V, int64_t d, int64_t K, void* stream) {
  PGN_CHECK_ARG(head_shape_ok(n, V, d, K));
  PGN_CHECK_ARG(h && W && aligned(h) && aligned(W) && (dh || dW) && aligned(dh) && aligned(dW));
  PGN_CHECK_ARG(!(g_ce || g_lse) || lse);
  PGN_CHECK_ARG(!g_ce || y);
  PGN_CHECK_ARG(!g_kd || (K > 0 && lse_t && psum && entry && p && zl));
  PGN_CHECK_ARG(g_ce || g_lse || g_kd);
  PGN_CHECK_ARG(tau > 0.f && tau < INFINITY);
  PGN_CHECK_ARG(workspace && aligned(workspace) && workspace_bytes >= pragnosia_head_bwd_workspace_bytes(n, V, d));
  hipStream_t st = (hipStream_t)stream;
  const Plan pl = plan(n, V);
  const bool ce = g_ce || g_lse;
  const int second = ce && g_kd && tau != 1.f;
  const float scale0 = ce ? 1.f : 1.f / tau, scale1 = 1.f / tau;
  const BwdIn in{g_ce, g_lse, g_kd, ce ? lse : nullptr, lse_t, psum, y, tau};
  const Operand ho{(const __bf16*)h, d, n}, Wo{(const __bf16*)W, d, V};
  __bf16* dl = (__bf16*)workspace;
  float* acc = (float*)(dl + pl.n_pad * pl.v_piece);
  hipError_t e = pgn_lds_limit((const void*)head_dlogits<1>, kGemmLds);
  if (e == hipSuccess) e = pgn_lds_limit((const void*)head_dlogits<2>, kGemmLds);
  if (e == hipSuccess) e = pgn_lds_limit((const void*)head_grads, kGemmLds);
  if (e != hipSuccess) return (int)e;
  const int64_t ty = pl.n_pad / kGemmTile, td = round_up(d, kGemmTile) / kGemmTile;
  for (int64_t q = 0; q < pl.pieces; ++q) {
    const int64_t v0 = q * pl.v_piece, words = std::min(pl.v_piece, V - v0), ld = round_up(words, kGemmTile);
    const int64_t items = ld / kGemmTile * ty;
    if (second)
      hipLaunchKernelGGL(head_dlogits<2>, dim3(xcd_grid(items)), dim3(kGemmThreads), kGemmLds, st, ho, Wo, in, scale0,
                         scale1, dl, ld, v0, d);
    else
      hipLaunchKernelGGL(head_dlogits<1>, dim3(xcd_grid(items)), dim3(kGemmThreads), kGemmLds, st, ho, Wo, in, scale0,
                         scale1, dl, ld, v0, d);
    if (g_kd)
      hipLaunchKernelGGL(head_entry_dl, dim3((unsigned)((n * K + 255) / 256)), dim3(256), 0, st, in, entry, p, zl, dl,
                         ld, v0, n, V, K);
    GradArgs ga;
    ga.dl_rows = ga.dl_words = Operand{dl, ld, pl.n_pad};
    ga.W = Operand{Wo.p + v0 * d, d, words};
    ga.h = ho;
    ga.n = n, ga.d = d, ga.words = words, ga.n_pad = pl.n_pad, ga.ld = ld;
    ga.dh = (__bf16*)dh, ga.dh_acc = acc, ga.first = q == 0, ga.last = q == pl.pieces - 1;
    ga.dW = dw_f32 ? (void*)((float*)dW + v0 * d) : (void*)((__bf16*)dW + v0 * d), ga.dw_f32 = dw_f32;
    ga.items_h = dh ? ty * td : 0, ga.items_w = dW ? ld / kGemmTile * td : 0;
    hipLaunchKernelGGL(head_grads, dim3(xcd_grid(ga.items_h + ga.items_w)), dim3(kGemmThreads), kGemmLds, st, ga);
  }
  PGN_RETURN_LAUNCH();
}
