// Losses of a head l = h W^T over a vocabulary, and their gradients, with no logits kept: cross entropy of labels and
// distillation from a teacher's top logits (formulas at pragnosia_head_fwd).
//
// Forward: each tile of 256 words x 256 tokens is one matrix product whose logits stay in the accumulators; every wave
// reduces its 128 words per token to a maximum and a sum of exponentials (two, where the cross entropy and a softened
// distillation loss share the pass), in fp32. A last kernel joins a row's pieces. The operands are swapped (words are
// the product's rows), so a token's words lie in one lane's registers and the reduction is two lane exchanges a token.
//
// Backward: the logits are formed again per piece of the vocabulary, turned into dl in the accumulators and rounded to
// bf16 (the operands' own precision: relative 2^-8 at most of each element, over a common scale, see RowInfo) into a
// workspace of the piece's columns; dh += dl W and dW = dl^T h are products over it.
//
// Bounds. All large products here run at the card's power limit: on these operands' random values the clock falls to
// about 1.8 GHz (2.3 on zeros), and taking stalls out of a kernel lowers the clock instead of the time. At 8192 tokens
// x 8192 words x 768 (103 GFLOP a product): head_logits 94 us (1.1 PFLOP/s; the library's plain product of these
// operands 92), head_dlogits 107 (the second exponential pass and 134 MB written), head_grads 165 for its two products
// (1.25 PFLOP/s; the library's two 296). Few tokens are bound by launches: at 64 tokens every kernel takes 4 to 15 us.
#include <algorithm>

#include "../include/pragnosia_lm.h"
#include "gemm_tile.h"

using namespace pgn;

namespace {

// Tiles of the logits (words x tokens), and of the gradients' products (columns of h or W x rows). A large one reaches
// the matrix cores' rate; smaller ones fill the chip where there are few tokens (choose_logits, choose_grads).
typedef Tile<8, 4, 2, 4, 2> Large;  // 256 x 256, 8 waves
typedef Tile<6, 4, 2, 4, 2> Wide;   // 192 x 256, 8 waves: four cover widths of 704 and 768 with less left over
typedef Tile<4, 4, 2, 2, 2> Mid;    // 128 x 128, 4 waves, two workgroups a compute unit
typedef Tile<2, 2, 2, 2, 4> Small;  // 64 x 64, 4 waves, two workgroups a compute unit
enum Kind { kLarge, kWide, kMid, kSmall };

struct KindInfo {
  int x, y, slots;    // tile, and workgroups that run at once
  float step, fixed;  // microseconds of a step of 64, and of a tile beside its steps, as measured on a full chip
};
constexpr KindInfo kLogitsKinds[] = {{Large::X, Large::Y, 256, 1.45f, 5.f},
                                     {Wide::X, Wide::Y, 256, 1.2f, 4.f},
                                     {Mid::X, Mid::Y, 512, 0.85f, 3.f},
                                     {Small::X, Small::Y, 512, 0.4f, 1.5f}};
constexpr KindInfo kGradKinds[] = {{Large::X, Large::Y, 256, 1.6f, 6.f},
                                   {Wide::X, Wide::Y, 256, 1.36f, 6.f},
                                   {Mid::X, Mid::Y, 512, 1.0f, 4.f}};

int64_t tiles(int64_t x, int64_t m) { return (x + m - 1) / m; }
int64_t round_up(int64_t x, int64_t m) { return tiles(x, m) * m; }

// The tile kind of the logits of n tokens and V words: the least time by rounds of tiles.
Kind choose_logits(int64_t n, int64_t V, int64_t d) {
  Kind best = kLarge;
  float least = INFINITY;
  for (Kind k : {kLarge, kWide, kMid, kSmall}) {
    const KindInfo& i = kLogitsKinds[k];
    const float t = (float)tiles(tiles(n, i.y) * tiles(V, i.x), i.slots) * (tiles(d, kGemmK) * i.step + i.fixed);
    if (t < least) least = t, best = k;
  }
  return best;
}

// The workspace of one piece's dl: about this many bytes at most (but 1024 words). It stays in the memory-side cache;
// half of it costs 12 - 18% more time, twice or four times gain under 1%.
constexpr int64_t kPieceBytes = (int64_t)144 << 20;

// How the gradients' products are laid out: the pieces of the vocabulary; the tile; the ranges that the contracted
// dimension is cut into (words for dh, tokens for dW), each a multiple of 64, so that few output tiles still fill the
// chip: the ranges' partial sums, fp32, are added in order by head_sum.
struct GradPlan {
  int64_t v_piece, pieces;
  Kind logits;        // the tile that forms dl
  int64_t n_pad, ld;  // dl's rows and pitch: whole tiles
  Kind kind;          // the products' tile
  int64_t len_h, split_h, len_w, split_w;
  int64_t dl_bytes, part_h, part_w;  // bytes of the workspace's three parts
};

// When `slots` workers have done n1 items of c1, then n2 of c2 <= c1, each taking the next as it comes free.
float makespan(int64_t n1, float c1, int64_t n2, float c2, int64_t slots) {
  const int64_t full = n1 / slots, rest = n1 - full * slots;
  const float at = full * c1, done = rest ? at + c1 : at;
  auto room = [&](float t) {
    return (slots - rest) * (int64_t)std::max(0.f, (t - at) / c2 + 1e-3f) +
           rest * (int64_t)std::max(0.f, (t - at - c1) / c2 + 1e-3f);
  };
  float lo = 0.f, hi = at + c1 + c2 * (n2 / slots + 1);
  for (int u = 0; u < 16; ++u) {
    const float mid = 0.5f * (lo + hi);
    (room(mid) >= n2 ? hi : lo) = mid;
  }
  return std::max(done, hi);
}

GradPlan search_grads(int64_t n, int64_t V, int64_t d) {
  GradPlan p;
  const int64_t most = std::max<int64_t>(1024, kPieceBytes / (2 * round_up(n, Large::Y))), count = tiles(V, most);
  p.logits = choose_logits(n, tiles(V, count), d);
  p.v_piece = count == 1 ? V : round_up(tiles(V, count), kLogitsKinds[p.logits].x);
  p.pieces = tiles(V, p.v_piece);
  p.n_pad = round_up(n, kLogitsKinds[p.logits].y);
  p.ld = round_up(p.v_piece, kLogitsKinds[p.logits].x);
  const int64_t words = std::min(V, p.v_piece), steps_h = tiles(words, kGemmK), steps_w = tiles(n, kGemmK);
  float least = INFINITY;
  for (Kind k : {kLarge, kWide, kMid}) {
    const KindInfo& i = kGradKinds[k];
    const int64_t tx = tiles(d, i.x), th = tx * tiles(n, i.y), tw = tx * tiles(words, i.y);
    for (int64_t len = 4; ; len *= 2) {  // steps of an item, at most
      const int64_t sh = tiles(steps_h, len), sw = tiles(steps_w, len);
      const int64_t lh = tiles(steps_h, sh), lw = tiles(steps_w, sw);
      const float ch = lh * i.step + i.fixed, cw = lw * i.step + i.fixed;
      float t = ch >= cw ? makespan(th * sh, ch, tw * sw, cw, i.slots) : makespan(tw * sw, cw, th * sh, ch, i.slots);
      // partial sums: written and read at about 4 bytes a picosecond, and a launch
      const float part = (sh > 1 ? 8.f * sh * n * d : 0.f) + (sw > 1 ? 8.f * sw * words * d : 0.f);
      if (part > 0.f) t += part * 0.25e-6f + 3.f;
      if (sh <= 64 && sw <= 64 && t < least) {
        least = t;
        p.kind = k;
        p.len_h = lh * kGemmK, p.split_h = tiles(steps_h, lh), p.len_w = lw * kGemmK, p.split_w = tiles(steps_w, lw);
      }
      if (sh == 1 && sw == 1) break;
    }
  }
  p.dl_bytes = round_up(p.n_pad * p.ld * 2, 256);
  p.part_h = p.split_h > 1 || p.pieces > 1 ? p.split_h * n * d * 4 : 0;
  p.part_w = p.split_w > 1 ? p.split_w * words * d * 4 : 0;
  return p;
}

// (The search takes microseconds of the host; a program's sizes repeat.)
GradPlan choose_grads(int64_t n, int64_t V, int64_t d) {
  thread_local struct {
    int64_t n = 0, V = 0, d = 0;
    GradPlan plan;
  } last;
  if (last.n != n || last.V != V || last.d != d) last = {n, V, d, search_grads(n, V, d)};
  return last.plan;
}

// Lane exchange of the groups of 16: the maximum, and the sum, over a column's four lane groups, in every one of them.
PGN_DEVICE float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
PGN_DEVICE float column_sum(float x) { return swap_add<32>(swap_add<16>(x, x), swap_add<16>(x, x)); }

// ---------------------------------------------------------------------------------------------------------------
// The teacher's distribution over its entries, a wave a row; bound by latency (8192 rows of 32 entries: 7 us). A
// repeated id's probabilities are added into its first entry, the others leave the list, so that every later kernel
// meets an id once, and the row's sum of p log p is that of the words (summed again where an id repeats).
constexpr int kMaxEntries = 1024;
constexpr float kTauLeast = 0x1p-10f;
constexpr int64_t kSliceBytes = (int64_t)2 << 20;

__global__ __launch_bounds__(256) void head_teacher(const int64_t* __restrict__ ids, const float* __restrict__ z,
                                                    float inv_tau, int32_t* __restrict__ entry,
                                                    float* __restrict__ p, float* __restrict__ psum,
                                                    float* __restrict__ ent, float* __restrict__ zl, int64_t n,
                                                    int64_t V, int K) {
  extern __shared__ __align__(16) unsigned char smem[];  // a wave's ids and probabilities
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * 4 + w;
  if (row >= n) return;
  const int K4 = (K + 3) / 4 * 4;
  int32_t* const id_of = reinterpret_cast<int32_t*>(smem) + w * 2 * K4;
  float* const p_of = reinterpret_cast<float*>(id_of + K4);
  ids += row * K, z += row * K, entry += row * K, p += row * K, zl += row * K;
  float m = -INFINITY;
  bool nan = false;
  for (int k = l; k < K; k += 64) {
    const int64_t id = ids[k];
    const bool on = id >= 0 && id < V;
    const float x = on ? z[k] : -INFINITY;
    id_of[k] = on ? (int32_t)id : -1;
    p_of[k] = x;
    m = fmaxf(m, x);
    nan = nan || x != x;
  }
  for (int o = 1; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
  if (__ballot(nan)) m = NAN;  // (a maximum passes over it; the row's probabilities and loss are NaN)
  const bool some = m != -INFINITY;
  float sum = 0.f;
  for (int k = l; k < K; k += 64)
    if (some && id_of[k] >= 0) sum += expf((p_of[k] - m) * inv_tau);
  for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
  const float inv = some ? 1.f / sum : 0.f, log_sum = some ? logf(sum) : 0.f;
  float e = 0.f;
  for (int k = l; k < K; k += 64) {
    const float x = (p_of[k] - m) * inv_tau;
    const bool on = some && id_of[k] >= 0;
    const float pk = on ? expf(x) * inv : 0.f;
    if (!on) id_of[k] = -1;
    p_of[k] = pk;
    if (pk != 0.f) e += pk * (x - log_sum);
  }
  if (l < K4 - K) id_of[K + l] = -1;
  // (the lists are the wave's own: its LDS operations are in order)
  __builtin_amdgcn_wave_barrier();
  bool repeats = false;
  for (int k = l; k < K + l; k += 64) {  // every lane takes part in every turn
    const int id = k < K ? id_of[k] : -1;
    float pk = k < K ? p_of[k] : 0.f;
    int earlier = 0, equal = 0;
#pragma unroll 4
    for (int j = 0; j < K4; j += 4) {
      const i32x4 o = *reinterpret_cast<const i32x4*>(id_of + j);
#pragma unroll
      for (int u = 0; u < 4; ++u) equal += o[u] == id;
    }
    if (__ballot(id >= 0 && equal > 1)) {  // a repeated id
      repeats = true;
      float all = 0.f;
      for (int j = 0; j < K; ++j)
        if (id_of[j] == id) {
          all += p_of[j];
          earlier += j < k;
        }
      pk = earlier == 0 ? all : 0.f;
    }
    if (k < K) {
      entry[k] = earlier == 0 ? id : -1;
      p[k] = id >= 0 ? pk : 0.f;
      if (id < 0 || earlier > 0) zl[k] = 0.f;  // (the others are head_entry_logits')
    }
  }
  if (repeats) {  // (p as this lane has just written it)
    e = 0.f;
    for (int k = l; k < K; k += 64)
      if (p[k] != 0.f) e += p[k] * logf(p[k]);
  }
  for (int o = 1; o < 64; o *= 2) e += __shfl_xor(e, o);
  if (l == 0) {
    psum[row] = some ? 1.f : 0.f;
    ent[row] = e;
  }
}

// s + a . b of eight bf16 pairs, in fp32 two products at a time.
PGN_DEVICE float dot8(bf16x8 a, bf16x8 b, float s) {
  typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    s = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a[2 * i], a[2 * i + 1]}, bf16x2{b[2 * i], b[2 * i + 1]}, s, false);
  return s;
}

// The student's logits of the teacher's entries, zl[i][k] = h_i . W_entry: 16 lanes a row and slice of the vocabulary,
// two entries at a time. Bound by the rows of W fetched (n K d values). An XCD takes every eighth slice, all rows of
// one before the next, so that the words' rows stay in its L2 (a slice is at most 2 MB): 8192 rows of 32 entries, 768
// wide, 31 us, 13 TB/s of rows; without slices, a wave a row, 44.
template <int CHUNKS>  // 128 values of d each, h's held in registers; 0: any d
__global__ __launch_bounds__(256) void head_entry_logits(const __bf16* __restrict__ h, const __bf16* __restrict__ W,
                                                         const int32_t* __restrict__ entry, float* __restrict__ zl,
                                                         int64_t n, int d, int K, int blocks, int slice) {
  constexpr int R = CHUNKS > 0 ? CHUNKS : 1;
  const int l = threadIdx.x & 63, q = l >> 4, j = l & 15;
  const int turn = blockIdx.x / kXcdCount / blocks, block = blockIdx.x / kXcdCount % blocks;
  const int lo = (turn * kXcdCount + blockIdx.x % kXcdCount) * slice;
  const int64_t row = (int64_t)block * 16 + (threadIdx.x >> 4);
  const bool live = row < n;
  const int64_t at = live ? row : n - 1;
  const __bf16* hr = h + at * d;
  entry += at * K, zl += at * K;
  bf16x8 x[R];
  if constexpr (CHUNKS > 0) {
#pragma unroll
    for (int c = 0; c < R; ++c)
      x[c] = 8 * j + 128 * c < d ? *reinterpret_cast<const bf16x8*>(hr + 8 * j + 128 * c) : bf16x8{};
  }
  for (int k0 = 0; k0 < K; k0 += 64) {
    // the row's entries within the slice, a bit each
    unsigned long long left = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int k = k0 + 16 * c + j, e = live && k < K ? entry[k] : -1;
      left |= (__ballot(e >= lo && e - lo < slice) >> (16 * q) & 0xffffull) << (16 * c);
    }
    while (__ballot(left != 0)) {
      int k[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        k[u] = left ? k0 + __ffsll((long long)left) - 1 : -1;
        left &= left - 1;
      }
      const __bf16* wr[2];
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u) wr[u] = W + (int64_t)(k[u] >= 0 ? entry[k[u]] : lo) * d + 8 * j;
      if constexpr (CHUNKS > 0) {
        bf16x8 w[2][R];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int c = 0; c < R; ++c)
            w[u][c] = 8 * j + 128 * c < d ? *reinterpret_cast<const bf16x8*>(wr[u] + 128 * c) : bf16x8{};
#pragma unroll
        for (int c = 0; c < R; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) s[u] = dot8(x[c], w[u][c], s[u]);
      } else {
        for (int c = 0; 8 * j + c < d; c += 128) {
          const bf16x8 a = *reinterpret_cast<const bf16x8*>(hr + 8 * j + c);
#pragma unroll
          for (int u = 0; u < 2; ++u) s[u] = dot8(a, *reinterpret_cast<const bf16x8*>(wr[u] + c), s[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = group_sum<16>(s[u]);
        if (j == 0 && k[u] >= 0) zl[k[u]] = s[u];
      }
    }
  }
}

struct FwdOut {
  float *m, *s0, *s1;  // pieces x n: maximum of l, sums of exp(scale0 (l - m)) and exp(scale1 (l - m))
  float* label;        // n: the label's logit (written only where the label is in range)
};

// Tiles of logits, reduced: a wave's words are one piece of its tokens' rows. The exponentials and maxima of a tile
// are 7% of its cycles, its twelve steps at d = 768 the rest. NEXP sums of exponentials, of scale0 l and scale1 l. y:
// labels, or null.
template <class C, int NEXP>
__global__ __launch_bounds__(C::kThreads) void head_logits(Operand h, Operand W, const int64_t* __restrict__ y,
                                                           float scale0, float scale1, FwdOut out, int64_t d) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int64_t n = h.rows;
  const int tx = (int)((W.rows + C::X - 1) / C::X), ty = (int)((n + C::Y - 1) / C::Y);
  const XcdRun run = xcd_run(tx * ty);
  if (run.first >= run.end) return;
  constexpr int kWords = 16 * C::NA;
  const float c0 = scale0 * kLog2e, c1 = scale1 * kLog2e;
  gemm_tiles<C, 8, 0>(
      W, h, d, y, n, run, smem, [&](int item, int& ix, int& iy) { band_tile(item, tx, ty, ix, iy); },
      [&](f32x4(&acc)[C::NA][C::NB], int64_t x0, int64_t y0, const unsigned char* info) {
        const WaveIdx t = wave_idx_opaque();  // (its addresses are made here, not held in registers over the steps)
        const int wx = t.w % C::WX, wy = t.w / C::WX;
        const int64_t v0 = x0 + kWords * wx;
        if (v0 + kWords > W.rows) {
#pragma unroll
          for (int a = 0; a < C::NA; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (v0 + 16 * a + 4 * t.g + r >= W.rows)
#pragma unroll
                for (int b = 0; b < C::NB; ++b) acc[a][b][r] = -INFINITY;
        }
        const int64_t piece = (v0 / kWords) * n;
#pragma unroll
        for (int b = 0; b < C::NB; ++b) {
          const int local = 16 * C::NB * wy + 16 * b + t.i;
          const int64_t row = y0 + local;
          if (y != nullptr) {
            const int64_t label = reinterpret_cast<const int64_t*>(info)[local], at = label - v0;
            const bool here = row < n && at >= 0 && at < kWords && label < W.rows;
            if (__ballot(here)) {
              const int own = here ? (int)at - 4 * t.g : -1;
#pragma unroll
              for (int a = 0; a < C::NA; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (own == 16 * a + r) out.label[row] = acc[a][b][r];
            }
          }
          float m = acc[0][b][0];
#pragma unroll
          for (int a = 0; a < C::NA; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[a][b][r]);
          m = column_max(m);
          const float base = m > -INFINITY ? m : 0.f, b0 = base * c0, b1 = base * c1;
          float s0 = 0.f, s1 = 0.f;
#pragma unroll
          for (int a = 0; a < C::NA; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              s0 += exp2_hw(__builtin_fmaf(acc[a][b][r], c0, -b0));
              if constexpr (NEXP == 2) s1 += exp2_hw(__builtin_fmaf(acc[a][b][r], c1, -b1));
            }
          s0 = column_sum(s0);
          if constexpr (NEXP == 2) s1 = column_sum(s1);
          if (t.g == 0 && row < n) {
            out.m[piece + row] = m;
            out.s0[piece + row] = s0;
            if constexpr (NEXP == 2) out.s1[piece + row] = s1;
          }
        }
      });
}

// Rows' pieces joined: R rows a workgroup, T = 256 / R threads a row (thread R q + r: every T-th piece of row r from
// q), each in one pass with a running maximum. Few rows take more threads each (7 rows of 256 pieces: 9 us with 16
// threads a row, 4 with 64; 8192 rows of 64 pieces: 5.5 us with 16).
struct JoinArgs {
  const int64_t* y;
  float *ce, *lse;
  const float *ent, *psum, *p, *zl;
  float *kd, *lse_t;
  float tau, scale0, scale1;
  int second;
  int64_t pieces, n, V, K;
};

template <int R>
__global__ __launch_bounds__(256) void head_join(FwdOut in, JoinArgs j) {
  constexpr int T = 256 / R;
  __shared__ float part[4][256];
  const int tid = threadIdx.x, r = tid % R, q = tid / R;
  const int64_t n = j.n, row = min((int64_t)blockIdx.x * R + r, n - 1);
  float m = -INFINITY, s0 = 0.f, s1 = 0.f;
#pragma unroll 4
  for (int64_t k = q; k < j.pieces; k += T) {
    const float mk = in.m[k * n + row], a0 = in.s0[k * n + row], a1 = j.second ? in.s1[k * n + row] : 0.f;
    const float top = fmaxf(m, mk), base = top > -INFINITY ? top : 0.f;
    s0 = s0 * expf((m - base) * j.scale0) + a0 * expf((mk - base) * j.scale0);
    if (j.second) s1 = s1 * expf((m - base) * j.scale1) + a1 * expf((mk - base) * j.scale1);
    m = top;
  }
  // the row's sum over the entries: consecutive threads take consecutive entries
  float dot = 0.f;
  if (j.K > 0) {
    const int64_t at = min((int64_t)blockIdx.x * R + tid / T, n - 1) * j.K;
    for (int64_t k = tid % T; k < j.K; k += T) {
      const float pk = j.p[at + k];
      if (pk != 0.f) dot += pk * j.zl[at + k];
    }
  }
  part[0][tid] = m, part[1][tid] = s0, part[2][tid] = s1, part[3][tid] = dot;
  for (int half = T / 2; half > 0; half /= 2) {
    __syncthreads();
    if (q < half) {
      const float mk = part[0][tid + half * R], top = fmaxf(m, mk), base = top > -INFINITY ? top : 0.f;
      const float f0 = expf((m - base) * j.scale0), g0 = expf((mk - base) * j.scale0);
      s0 = s0 * f0 + part[1][tid + half * R] * g0;
      if (j.second)
        s1 = s1 * expf((m - base) * j.scale1) + part[2][tid + half * R] * expf((mk - base) * j.scale1);
      m = top;
      part[0][tid] = m, part[1][tid] = s0, part[2][tid] = s1;
    }
    if (tid % T < half) part[3][tid] += part[3][tid + half];
  }
  __syncthreads();
  if (q != 0 || (int64_t)blockIdx.x * R + r >= n) return;
  dot = part[3][r * T];
  const float l0 = m * j.scale0 + logf(s0), l1 = j.second ? m * j.scale1 + logf(s1) : l0;
  if (j.y != nullptr) {
    const int64_t label = j.y[row];
    j.lse[row] = l0;
    j.ce[row] = label >= 0 && label < j.V ? l0 - in.label[row] : 0.f;
  }
  if (j.K > 0) {
    j.lse_t[row] = l1;
    j.kd[row] = j.psum[row] > 0.f ? j.tau * j.tau * (j.ent[row] - dot / j.tau + l1) : 0.f;
  }
}

// ---------------------------------------------------------------------------------------------------------------
struct BwdIn {
  const float *g_ce, *g_lse, *g_kd, *lse, *lse_t, *psum;
  const int64_t* y;
  float tau;
};

// What dl takes of a row, over the common scale G: dl / G = w0 exp(l scale0 - l0) + w1 exp(l scale1 - l1) -
// gc [v = label], the exponents in base 2; zero where not live.
//
// G is the largest of the rows' gradients of the cross entropy (of the distillation loss, where there is no label: a
// teacher's probabilities are no constants, and round at random), over the rows that have a label (a teacher). A mean's
// rows all have the same weight w, and most of a row's gradient is its label's -w (1 - p) with a small p: rounded as it
// stands, every row would carry the same relative error, that of w's bf16 (up to 2^-8). Over G the weights are 1, the
// label's element is within 2^-9 and mostly much nearer, and the products are multiplied by G in fp32. Where another
// loss's weights are more than 2^64 times as large, or overflow with tau, G is 2^-64 of the largest: neither the large
// ones overflow over it nor are those of a token that has only the small ones lost.
struct RowInfo {
  float w0, l0, w1, l1, gc;
  int32_t label, live, unused;
};

struct RowWeights {
  float ce, kd, gc;  // kd over g
  int64_t label;     // -1: none
};

PGN_DEVICE RowWeights row_weights(const BwdIn& in, int64_t row, int64_t V, float g) {
  RowWeights r;
  r.label = in.y != nullptr ? in.y[row] : -1;
  if (r.label < 0 || r.label >= V) r.label = -1;
  r.gc = r.label >= 0 && in.g_ce != nullptr ? in.g_ce[row] : 0.f;
  r.ce = r.gc + (in.g_lse != nullptr ? in.g_lse[row] : 0.f);
  r.kd = 0.f;
  if (in.g_kd != nullptr && in.psum[row] != 0.f) {
    const float kd = in.g_kd[row], x = kd * in.tau;
    r.kd = fabsf(x) < INFINITY ? x / g : kd / g * in.tau;
  }
  return r;
}

// The largest magnitude, among the rows of [a, b) that this thread of 1024 meets (a: a multiple of four), of the
// gradient of the cross entropy (which 0: of rows with a label), the distillation loss (1: of rows with a teacher) or
// the log-denominator (2). A row whose loss is a constant 0 takes no part: its weight, of any size, is no weight of dl's.
PGN_DEVICE float thread_max(const BwdIn& in, int which, int64_t a, int64_t b, int64_t V, int tid) {
  typedef int64_t i64x4_any __attribute__((__vector_size__(32), __aligned__(8)));
  typedef float f32x4_any __attribute__((__vector_size__(16), __aligned__(4)));
  const float* x = which == 0 ? in.g_ce : which == 1 ? in.g_kd : in.g_lse;
  float g = 0.f;
  auto take = [&](float v, int64_t label, float some) {
    g = fmaxf(g, label >= 0 && label < V && some != 0.f ? fabsf(v) : 0.f);
  };
#pragma unroll 2
  for (int64_t k = a + 4 * tid; k + 4 <= b; k += 4096) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(x + k);
    i64x4_any label{};
    f32x4_any some{1.f, 1.f, 1.f, 1.f};
    if (which == 0) label = *reinterpret_cast<const i64x4_any*>(in.y + k);
    if (which == 1) some = *reinterpret_cast<const f32x4_any*>(in.psum + k);
#pragma unroll
    for (int u = 0; u < 4; ++u) take(v[u], label[u], some[u]);
  }
  const int64_t k = b - 1 - tid;
  if (tid < (b - a) % 4) take(x[k], which == 0 ? in.y[k] : 0, which == 1 ? in.psum[k] : 1.f);
  return g;
}

// The three losses' maxima over the workgroup's 1024 threads (by place: two losses' gradients may be one array): of
// rows [a, b), or of the `parts` triples of `part` where there are any.
PGN_DEVICE void group_max(const BwdIn& in, const float* __restrict__ part, int parts, int64_t a, int64_t b, int64_t V,
                          float (&v)[3]) {
  __shared__ float most[3][16];
  const int tid = threadIdx.x;
#pragma unroll
  for (int which = 0; which < 3; ++which) {
    const bool there = (which == 0 ? in.g_ce : which == 1 ? in.g_kd : in.g_lse) != nullptr;
    v[which] = 0.f;
    if (there && parts == 0) v[which] = thread_max(in, which, a, b, V, tid);
    if (tid < parts) v[which] = part[3 * tid + which];
    for (int o = 1; o < 64; o *= 2) v[which] = fmaxf(v[which], __shfl_xor(v[which], o));
    if ((tid & 63) == 0) most[which][tid >> 6] = v[which];
  }
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 3; ++which)
    for (int k = 0; k < 16; ++k) v[which] = fmaxf(v[which], most[which][k]);
}

// Rows' maxima by workgroup, for head_rows over many rows: part[3 b ..], `each` rows a workgroup.
__global__ __launch_bounds__(1024) void head_most(BwdIn in, float* __restrict__ part, int64_t n, int64_t V,
                                                  int64_t each) {
  float v[3];
  group_max(in, nullptr, 0, blockIdx.x * each, min(n, (int64_t)(blockIdx.x + 1) * each), V, v);
  if (threadIdx.x < 3) part[3 * blockIdx.x + threadIdx.x] = threadIdx.x == 0 ? v[0] : threadIdx.x == 1 ? v[1] : v[2];
}

// Rows past which the maxima are found by a launch of their own, as every workgroup of head_rows would read all rows'
// gradients and labels (32768 rows: 9.0 us in one launch, 8.5 in two; 65536: 13.6, 8.6; 2^20: 161, 18).
constexpr int64_t kManyRows = (int64_t)1 << 15;
constexpr int64_t kMostBytes = 256 * 3 * sizeof(float);

// Every workgroup finds G itself (4.5 us at 8192 rows, 5.6 with two losses: launch and latency), from all rows'
// gradients (at most 256 workgroups, `each` rows of their own); *scale = G. Past kManyRows rows, from `parts` maxima of
// head_most's.
__global__ __launch_bounds__(1024) void head_rows(BwdIn in, int second, RowInfo* __restrict__ rows,
                                                  float* __restrict__ scale, const float* __restrict__ part, int parts,
                                                  int64_t n, int64_t V, int64_t each) {
  const int tid = threadIdx.x;
  float v[3];
  group_max(in, part, parts, 0, n, V, v);
  float g = 0.f, all = 0.f, raw = 0.f;
#pragma unroll
  for (int which = 0; which < 3; ++which) {
    if (!(v[which] < INFINITY)) continue;
    raw = fmaxf(raw, v[which]);
    const float x = which == 1 ? v[which] * in.tau : v[which];
    if (g == 0.f) g = x;
    all = fmaxf(all, x);
  }
  if (!(all <= g * 0x1p64f && g < INFINITY)) g = raw * 0x1p-64f;
  if (g == 0.f) g = 1.f;
  if (blockIdx.x == 0 && tid == 0) *scale = g;
  const int64_t end = min(n, (int64_t)(blockIdx.x + 1) * each);
  for (int64_t row = blockIdx.x * each + tid; row < end; row += 1024) {
    const RowWeights r = row_weights(in, row, V, g);
    RowInfo o{};
    o.label = (int32_t)r.label;
    o.gc = r.gc / g;
    o.w0 = r.ce / g + (second ? 0.f : r.kd);
    o.w1 = r.kd;
    o.l0 = (in.lse != nullptr ? in.lse[row] : in.lse_t[row]) * kLog2e;
    o.l1 = second ? in.lse_t[row] * kLog2e : 0.f;
    o.live = r.ce != 0.f || r.kd != 0.f || r.gc != 0.f;
    rows[row] = o;
  }
}

// Two adjacent accumulator tiles (rows 0 .. 15 and 16 .. 31 of a 32-row block; lane (i, g) holds rows 4 g .. 4 g + 3
// of column i of both) rounded to bf16, exchanged between lane groups so that a lane ends with eight consecutive rows
// of its column, first_of(g) ..: one 16-byte store, 64 bytes a column.
PGN_DEVICE int first_of(int g) { return 16 * (g & 1) + 8 * (g >> 1); }
PGN_DEVICE bf16x8 eight_rows(f32x4 lo, f32x4 hi) {
  const i32x2 x = __builtin_bit_cast(i32x2, to_bf16x4(lo)), y = __builtin_bit_cast(i32x2, to_bf16x4(hi));
  const auto p = __builtin_amdgcn_permlane16_swap((unsigned)x[0], (unsigned)y[0], false, false);
  const auto q = __builtin_amdgcn_permlane16_swap((unsigned)x[1], (unsigned)y[1], false, false);
  const unsigned p0 = p[0], p1 = p[1], q0 = q[0], q1 = q[1];
  return __builtin_bit_cast(bf16x8, i32x4{(int)p0, (int)q0, (int)p1, (int)q1});
}

// dl / G of a piece of the vocabulary: words v_begin .. v_begin + ld (whole tiles) of the workspace's n_pad rows
// (likewise). Word and token rows past the ends get zeros.
template <class C, int NEXP>
__global__ __launch_bounds__(C::kThreads) void head_dlogits(Operand h, Operand W, const RowInfo* __restrict__ rows,
                                                            float scale0, float scale1, __bf16* __restrict__ dl,
                                                            int64_t ld, int64_t v_begin, int64_t n_pad, int64_t d) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int64_t words = min(ld, W.rows - v_begin);
  const int tx = (int)(ld / C::X), ty = (int)(n_pad / C::Y);
  const XcdRun run = xcd_run(tx * ty);
  if (run.first >= run.end) return;
  const float e0 = scale0 * kLog2e, e1 = scale1 * kLog2e;
  const Operand Wp{W.p + v_begin * W.ld, W.ld, words};
  gemm_tiles<C, sizeof(RowInfo), C::NB * C::NA / 2>(
      Wp, h, d, rows, h.rows, run, smem, [&](int item, int& ix, int& iy) { band_tile(item, tx, ty, ix, iy); },
      [&](f32x4(&acc)[C::NA][C::NB], int64_t x0, int64_t y0, const unsigned char* info) {
        const WaveIdx t = wave_idx_opaque();
        const int wx = t.w % C::WX, wy = t.w / C::WX;
        const int64_t c0 = x0 + 16 * C::NA * wx;
        const bool partial = c0 + 16 * C::NA > words;
#pragma unroll
        for (int b = 0; b < C::NB; ++b) {
          const int local = 16 * C::NB * wy + 16 * b + t.i;
          const RowInfo o = reinterpret_cast<const RowInfo*>(info)[local];
          const int at = o.label - (int)(v_begin + c0);
          const bool here = o.gc != 0.f && at >= 0 && at < 16 * C::NA, hit = __ballot(here) != 0;
          const int own = here ? at - 4 * t.g : -1;
#pragma unroll
          for (int a = 0; a < C::NA; ++a) {
            f32x4 x = acc[a][b];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float z = o.w0 * exp2_hw(__builtin_fmaf(x[r], e0, -o.l0));
              if constexpr (NEXP == 2) z += o.w1 * exp2_hw(__builtin_fmaf(x[r], e1, -o.l1));
              x[r] = o.live ? z : 0.f;
            }
            acc[a][b] = x;
          }
          if (hit) {
#pragma unroll
            for (int a = 0; a < C::NA; ++a)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (own == 16 * a + r) acc[a][b][r] -= o.gc;
          }
          if (partial) {
#pragma unroll
            for (int a = 0; a < C::NA; ++a)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (c0 + 16 * a + 4 * t.g + r >= words) acc[a][b][r] = 0.f;
          }
        }
#pragma unroll
        for (int b = 0; b < C::NB; ++b) {
          __bf16* p = dl + (y0 + 16 * C::NB * wy + 16 * b + t.i) * ld + c0 + first_of(t.g);
#pragma unroll
          for (int a = 0; a < C::NA; a += 2)
            *reinterpret_cast<bf16x8*>(p + 16 * a) = eight_rows(acc[a][b], acc[a + 1][b]);
        }
      });
}

// dl / G at the teacher's entries, whole: a thread an entry, from the fp32 logit, so rounded once. Scattered two-byte
// stores: 6 us for 8192 x 32.
__global__ __launch_bounds__(256) void head_entry_dl(BwdIn in, const float* __restrict__ scale,
                                                     const int32_t* __restrict__ entry, const float* __restrict__ p,
                                                     const float* __restrict__ zl, __bf16* __restrict__ dl, int64_t ld,
                                                     int64_t v_begin, int64_t words, int64_t n, int64_t V, int64_t K) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n * K) return;
  const int64_t row = e / K;
  const int v = entry[e];
  if (v < v_begin || v >= v_begin + words) return;
  const float g = *scale;
  const RowWeights r = row_weights(in, row, V, g);
  float x = 0.f;
  if (r.ce != 0.f || r.kd != 0.f || r.gc != 0.f) {
    const float l = zl[e];
    if (r.kd != 0.f) x = r.kd * (expf(l / in.tau - in.lse_t[row]) - p[e]);  // (p may be NaN where the weight is zero)
    if (r.ce != 0.f) x += r.ce / g * expf(l - in.lse[row]);
    if (r.label == v) x -= r.gc / g;
  }
  dl[row * ld + (v - v_begin)] = (__bf16)x;
}

// dh = G (dl / G) W over a piece and dW = G (dl / G)^T h of the piece, in one launch; either whole, or as fp32 partial
// sums by range of the contracted dimension. One launch, so that neither's last tiles leave the chip idle: at 8192 x
// 8192 x 768 it is 256 workgroups of 192 x 256 for 256 compute units.
struct GradSide {
  int64_t rows, k, len, split;  // output rows; contracted length, its ranges
  void* out;                    // rows x d, where one range is all
  float* part;                  // split x rows x d
  int f32, add;                 // out's type; whether part holds earlier pieces' sums
};
struct GradArgs {
  Operand dl, W, h;  // dl by rows (n_pad); W's rows of the piece
  int64_t d;
  GradSide side[2];  // dh, dW
  const float* scale;  // G
  int first;           // the side whose items are longer, launched first
};

template <class C>
__global__ __launch_bounds__(C::kThreads) void head_grads(GradArgs q) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int64_t tx = (q.d + C::X - 1) / C::X;
  // each XCD takes a contiguous eighth of the first side's items, then of the second's
  int which = q.first;
  int64_t j = blockIdx.x / kXcdCount;
  for (int u = 0; u < 2; ++u, which ^= 1) {
    const GradSide& s = q.side[which];
    const int64_t items = s.out == nullptr ? 0 : tx * ((s.rows + C::Y - 1) / C::Y) * s.split;
    const int64_t per = (items + kXcdCount - 1) / kXcdCount;
    if (j < per) {
      const int64_t item = blockIdx.x % kXcdCount * per + j;
      if (item >= items) return;
      const int64_t range = item / (items / s.split), tile = item - range * (items / s.split), iy = tile / tx;
      const int64_t x0 = (tile - iy * tx) * C::X, y0 = iy * C::Y;
      const int64_t k0 = range * s.len, k1 = max(k0, min(s.k, k0 + s.len));
      f32x4 acc[C::NA][C::NB];
      if (which == 0)
        gemm_tile<C, true, false>(q.W, q.dl, x0, y0, k0, k1, smem, acc);
      else
        gemm_tile<C, true, true>(q.h, q.dl, x0, y0, k0, k1, smem, acc);
      const WaveIdx t = wave_idx();
      const int64_t c0 = x0 + 16 * C::NA * (t.w % C::WX);
      const float g = *q.scale;
#pragma unroll
      for (int b = 0; b < C::NB; ++b) {
#pragma unroll
        for (int a = 0; a < C::NA; ++a) acc[a][b] *= g;
        const int64_t row = y0 + 16 * C::NB * (t.w / C::WX) + 16 * b + t.i;
        if (s.part != nullptr || s.f32) {
          float* p = (s.part != nullptr ? s.part + (range * s.rows + row) * q.d : (float*)s.out + row * q.d);
#pragma unroll
          for (int a = 0; a < C::NA; ++a) {
            const int64_t c = c0 + 16 * a + 4 * t.g;
            if (row >= s.rows || c >= q.d) continue;
            f32x4 x = acc[a][b];
            if (s.part != nullptr && s.add) x += *reinterpret_cast<const f32x4*>(p + c);
            *reinterpret_cast<f32x4*>(p + c) = x;
          }
        } else {
#pragma unroll
          for (int a = 0; a < C::NA; a += 2) {
            const bf16x8 x = eight_rows(acc[a][b], acc[a + 1][b]);
            const int64_t c = c0 + 16 * a + first_of(t.g);
            if (row < s.rows && c < q.d) *reinterpret_cast<bf16x8*>((__bf16*)s.out + row * q.d + c) = x;
          }
        }
      }
      return;
    }
    j -= per;
  }
}

// out = the ranges' partial sums in order, four elements a thread.
__global__ __launch_bounds__(256) void head_sum(const float* __restrict__ part, void* __restrict__ out, int f32,
                                                int64_t split, int64_t count) {
  for (int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; e < count; e += (int64_t)gridDim.x * 1024) {
    f32x4 x = *reinterpret_cast<const f32x4*>(part + e);
    for (int64_t k = 1; k < split; ++k) x += *reinterpret_cast<const f32x4*>(part + k * count + e);
    if (f32)
      *reinterpret_cast<f32x4*>((float*)out + e) = x;
    else
      *reinterpret_cast<bf16x4*>((__bf16*)out + e) = to_bf16x4(x);
  }
}

// Logits kernels by tile kind: F<C> with the tile type.
template <class F>
auto by_kind(Kind k, F&& f) {
  return k == kLarge ? f(Large{}) : k == kWide ? f(Wide{}) : k == kMid ? f(Mid{}) : f(Small{});
}

int launch_sum(const float* part, void* out, int f32, int64_t split, int64_t count, hipStream_t st) {
  hipLaunchKernelGGL(head_sum, dim3((unsigned)std::min<int64_t>(tiles(count, 1024), 4096)), dim3(256), 0, st, part, out,
                     f32, split, count);
  return (int)hipGetLastError();
}

template <class C>
int launch_grads(const GradArgs& ga, hipStream_t st) {
  const hipError_t e = pgn_lds_limit((const void*)head_grads<C>, C::kLds);
  if (e != hipSuccess) return (int)e;
  int64_t groups = 0;
  for (const GradSide& s : ga.side)
    if (s.out != nullptr) groups += xcd_grid(tiles(ga.d, C::X) * tiles(s.rows, C::Y) * s.split);
  hipLaunchKernelGGL(head_grads<C>, dim3((unsigned)groups), dim3(C::kThreads), C::kLds, st, ga);
  return (int)hipGetLastError();
}

bool head_shape_ok(int64_t n, int64_t V, int64_t d, int64_t K) {
  return n > 0 && n <= (int64_t)1 << 24 && V > 0 && V <= (int64_t)1 << 24 && d > 0 && d % 8 == 0 && d <= 65536 &&
         K >= 0 && K <= kMaxEntries &&
         // launches of fewer than 2^32 threads; tiles counted in 32 bits
         n * K < (int64_t)1 << 31 && (K == 0 || tiles(n, 4) * (V * d >> 20) < (int64_t)1 << 23) &&
         tiles(n, Small::Y) * tiles(V, Small::X) < (int64_t)1 << 30 &&
         tiles(std::max(n, V), Mid::Y) * tiles(d, Mid::X) < (int64_t)1 << 21;
}

bool aligned(const void* p) { return ((uintptr_t)p % 16) == 0; }

// Pieces of a row's softmax: the words of a wave of the tile.
int64_t head_pieces(int64_t n, int64_t V, int64_t d) {
  const Kind k = choose_logits(n, V, d);
  return tiles(V, kLogitsKinds[k].x) * 2;
}
static_assert(Large::WX == 2 && Wide::WX == 2 && Mid::WX == 2 && Small::WX == 2, "two waves along the words");

}  // namespace

extern "C" int pragnosia_lm_abi_version(void) { return 1; }

extern "C" int64_t pragnosia_head_fwd_workspace_bytes(int64_t n, int64_t V, int64_t d, int64_t K) {
  if (!head_shape_ok(n, V, d, K)) return -1;
  return (3 * head_pieces(n, V, d) + 2) * n * (int64_t)sizeof(float);
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
  PGN_CHECK_ARG(tau >= kTauLeast && tau <= 1.f / kTauLeast);
  PGN_CHECK_ARG(workspace && aligned(workspace) && workspace_bytes >= pragnosia_head_fwd_workspace_bytes(n, V, d, K));
  hipStream_t st = (hipStream_t)stream;
  const int64_t pieces = head_pieces(n, V, d);
  float* f = (float*)workspace;
  const FwdOut out{f, f + pieces * n, f + 2 * pieces * n, f + 3 * pieces * n};
  float* ent = f + (3 * pieces + 1) * n;
  const Operand ho{(const __bf16*)h, d, n}, Wo{(const __bf16*)W, d, V};
  if (K > 0) {
    hipLaunchKernelGGL(head_teacher, dim3((unsigned)tiles(n, 4)), dim3(256), (unsigned)(4 * 8 * round_up(K, 4)), st,
                       ids, z, 1.f / tau, entry, p, psum, ent, zl, n, V, (int)K);
    // slices of at most 2 MB of W, eight a turn
    const int64_t turns = tiles(V * d * 2, kXcdCount * kSliceBytes), blocks = tiles(n, 16);
    const int64_t slice = tiles(V, kXcdCount * turns);
    const auto fn = d <= 512    ? head_entry_logits<4>
                    : d <= 768  ? head_entry_logits<6>
                    : d <= 1024 ? head_entry_logits<8>
                                : head_entry_logits<0>;
    hipLaunchKernelGGL(fn, dim3((unsigned)(kXcdCount * turns * blocks)), dim3(256), 0, st, ho.p, Wo.p, entry, zl, n,
                       (int)d, (int)K, (int)blocks, (int)slice);
  }
  const int second = y && K > 0 && tau != 1.f;
  const float scale0 = y ? 1.f : 1.f / tau, scale1 = 1.f / tau;
  const Kind kind = choose_logits(n, V, d);
  const int rc = by_kind(kind, [&](auto c) {
    typedef decltype(c) C;
    const auto fn = second ? head_logits<C, 2> : head_logits<C, 1>;
    const hipError_t e = pgn_lds_limit((const void*)fn, C::kLdsInfo);
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL(fn, dim3(xcd_grid(tiles(V, C::X) * tiles(n, C::Y), kLogitsKinds[kind].slots)), dim3(C::kThreads),
                       C::kLdsInfo, st, ho, Wo, y, scale0, scale1, out, d);
    return (int)hipGetLastError();
  });
  if (rc) return rc;
  const JoinArgs j{y, ce, lse, ent, psum, p, zl, kd, lse_t, tau, scale0, scale1, second, pieces, n, V, K};
  if (n <= 4096)
    hipLaunchKernelGGL(head_join<4>, dim3((unsigned)tiles(n, 4)), dim3(256), 0, st, out, j);
  else
    hipLaunchKernelGGL(head_join<16>, dim3((unsigned)tiles(n, 16)), dim3(256), 0, st, out, j);
  PGN_RETURN_LAUNCH();
}

extern "C" int64_t pragnosia_head_bwd_workspace_bytes(int64_t n, int64_t V, int64_t d) {
  if (!head_shape_ok(n, V, d, 0)) return -1;
  const GradPlan pl = choose_grads(n, V, d);
  return pl.dl_bytes + pl.part_h + pl.part_w + n * (int64_t)sizeof(RowInfo) + 16 + (n > kManyRows ? kMostBytes : 0);
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
  PGN_CHECK_ARG((g_ce || g_lse || g_kd) && aligned(g_ce) && aligned(g_lse) && aligned(g_kd));
  PGN_CHECK_ARG(tau >= kTauLeast && tau <= 1.f / kTauLeast);
  PGN_CHECK_ARG(workspace && aligned(workspace) && workspace_bytes >= pragnosia_head_bwd_workspace_bytes(n, V, d));
  hipStream_t st = (hipStream_t)stream;
  const GradPlan pl = choose_grads(n, V, d);
  const bool ce = g_ce || g_lse;
  const int second = ce && g_kd && tau != 1.f;
  const float scale0 = ce ? 1.f : 1.f / tau, scale1 = 1.f / tau;
  const BwdIn in{g_ce, g_lse, g_kd, ce ? lse : nullptr, lse_t, psum, y, tau};
  const Operand ho{(const __bf16*)h, d, n}, Wo{(const __bf16*)W, d, V};
  unsigned char* ws = (unsigned char*)workspace;
  __bf16* dl = (__bf16*)ws;
  float *part_h = (float*)(ws + pl.dl_bytes), *part_w = (float*)(ws + pl.dl_bytes + pl.part_h);
  RowInfo* rows = (RowInfo*)(ws + pl.dl_bytes + pl.part_h + pl.part_w);
  float* scale = (float*)(rows + n);
  const int64_t each = std::max<int64_t>(256, round_up(tiles(n, 256), 4));
  const int groups = (int)tiles(n, each), parts = n > kManyRows ? groups : 0;
  float* most = scale + 4;
  if (parts) hipLaunchKernelGGL(head_most, dim3(groups), dim3(1024), 0, st, in, most, n, V, each);
  hipLaunchKernelGGL(head_rows, dim3(groups), dim3(1024), 0, st, in, second, rows, scale, most, parts, n, V, each);
  for (int64_t q = 0; q < pl.pieces; ++q) {
    const int64_t v0 = q * pl.v_piece, words = std::min(pl.v_piece, V - v0);
    const int64_t ld = round_up(words, kLogitsKinds[pl.logits].x);
    int rc = by_kind(pl.logits, [&](auto c) {
      typedef decltype(c) C;
      const auto fn = second ? head_dlogits<C, 2> : head_dlogits<C, 1>;
      const hipError_t e = pgn_lds_limit((const void*)fn, C::kLdsInfo);
      if (e != hipSuccess) return (int)e;
      hipLaunchKernelGGL(fn, dim3(xcd_grid(ld / C::X * (pl.n_pad / C::Y), kLogitsKinds[pl.logits].slots)),
                         dim3(C::kThreads), C::kLdsInfo, st, ho, Wo, rows, scale0, scale1, dl, ld, v0, pl.n_pad, d);
      return (int)hipGetLastError();
    });
    if (rc) return rc;
    if (g_kd)
      hipLaunchKernelGGL(head_entry_dl, dim3((unsigned)tiles(n * K, 256)), dim3(256), 0, st, in, scale, entry, p, zl,
                         dl, ld, v0, words, n, V, K);
    void* dW_q = dW == nullptr ? nullptr
                               : dw_f32 ? (void*)((float*)dW + v0 * d) : (void*)((__bf16*)dW + v0 * d);
    GradArgs ga{Operand{dl, ld, pl.n_pad}, Operand{Wo.p + v0 * d, d, words}, ho, d,
                {{n, words, pl.len_h, pl.split_h, dh, pl.part_h ? part_h : nullptr, 0, q > 0},
                 {words, n, pl.len_w, pl.split_w, dW_q, pl.part_w ? part_w : nullptr, dw_f32, 0}},
                scale, pl.len_h >= pl.len_w ? 0 : 1};
    rc = pl.kind == kLarge ? launch_grads<Large>(ga, st)
                           : pl.kind == kWide ? launch_grads<Wide>(ga, st) : launch_grads<Mid>(ga, st);
    if (rc) return rc;
    if (dW && pl.part_w && (rc = launch_sum(part_w, dW_q, dw_f32, pl.split_w, words * d, st))) return rc;
  }
  if (dh && pl.part_h) {
    const int rc = launch_sum(part_h, dh, 0, pl.split_h, n * d, st);
    if (rc) return rc;
  }
  PGN_RETURN_LAUNCH();
}
