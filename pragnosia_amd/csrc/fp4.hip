// 4-bit weights for generation: rounding to e2m1 codes with a bf16 scale a group, reading back, and rows times such a
// weight with a LayerNorm before and bias, GELU and residual after (the dense layers of a decode step; formulas and
// layouts in include/pragnosia_gen.h).
//
// Codes lie as the matrix core takes them: a tile of 16 rows by 128 columns is one contiguous 1 KiB load, a lane's 16
// bytes the operands of four v_mfma_f32_16x16x32_bf16. Two codes become two bf16 numbers in one instruction
// (v_cvt_scalef32_pk_bf16_fp4), exactly, and a group's scale multiplies its fp32 sums: no weight is rounded again.
#include <algorithm>

#include "../include/pragnosia_gen.h"
#include "common.h"

namespace {

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u32x4;
typedef __attribute__((__vector_size__(2 * sizeof(unsigned short)))) unsigned short u16x2;

#define PGN_INLINE __attribute__((always_inline))  // of a lambda whose captured arrays have to stay in registers

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = 1024;

PGN_DEVICE unsigned bits_of(float x) { return __builtin_bit_cast(unsigned, x); }
PGN_DEVICE float float_of(unsigned u) { return __builtin_bit_cast(float, u); }
PGN_DEVICE float bf16_bits(unsigned u) { return float_of(u << 16); }

// Eight consecutive elements as they come from memory, and as fp32.
template <class T>
struct Raw;
template <>
struct Raw<float> {
  f32x4 a, b;
  PGN_DEVICE void load(const float* p) {
    a = reinterpret_cast<const f32x4*>(p)[0];
    b = reinterpret_cast<const f32x4*>(p)[1];
  }
  PGN_DEVICE void keep(bool k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = k ? a[e] : 0.f;
      b[e] = k ? b[e] : 0.f;
    }
  }
  PGN_DEVICE float get(int e) const { return e < 4 ? a[e & 3] : b[e & 3]; }
  // the largest absolute value, as its bits (their order is the values', a NaN above an infinity)
  PGN_DEVICE unsigned most() const {
    unsigned m = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, bits_of(get(e)) & 0x7fffffffu);
    return m;
  }
};
template <>
struct Raw<__bf16> {
  u32x4 a;
  PGN_DEVICE void load(const __bf16* p) { a = *reinterpret_cast<const u32x4*>(p); }
  PGN_DEVICE void keep(bool k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = k ? a[e] : 0u;
  }
  PGN_DEVICE float get(int e) const { return e & 1 ? float_of(a[e >> 1] & 0xffff0000u) : bf16_bits(a[e >> 1]); }
  PGN_DEVICE unsigned most() const {  // (two at a time)
    u16x2 m{0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, a[e] & 0x7fff7fffu));
    return (unsigned)max(m[0], m[1]) << 16;
  }
};

// ---------------------------------------------------------------------------------------------------------------
// rounding

// Maximum over the four lanes l % 16 + 16 h, in all of them.
PGN_DEVICE unsigned max_over_h(unsigned m) {
  const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  const unsigned m2 = a[0] > a[1] ? a[0] : a[1];
  const auto b = __builtin_amdgcn_permlane32_swap(m2, m2, false, false);
  return b[0] > b[1] ? b[0] : b[1];
}

// The code of w over the scale s, from the borders between codes: a border has at most 3 bits and s 8, so the products
// are exact. An equally near pair gives the even code.
PGN_DEVICE unsigned exact_code(float w, float s) {
  const float a = fabsf(w);
  const unsigned c = (a > 0.25f * s) + (a >= 0.75f * s) + (a > 1.25f * s) + (a >= 1.75f * s) + (a > 2.5f * s) +
                     (a >= 3.5f * s) + (a > 5.f * s);
  return c | (bits_of(w) >> 31) << 3;
}

// One wave a tile. A code is the hardware's rounding of w / s, to nearest even as the definition has it, of the quotient
// rounded once: a quotient that is not a border between codes does not round to one, as |w - t s| is at least a step of w for
// the exact product t s. Quotients come by a product with the reciprocal and one correction (correctly rounded, as the
// reciprocal is: all scales' mantissas were tried), where neither can leave the range; elsewhere by division and
// exact_code. Deciding the doubtful ones by exact_code instead (two quotients, a little too large and too small, that give
// different codes) took that path in every other wave of bf16 weights, which often lie on a border: 32768 x 4096 in 82 us.
// Bound by the weight's bytes where it is large (32768 x 4096 bf16 in 55 us, groups of 32: 6.2 TB/s, part of them from the
// memory-side cache), by a launch and one round of loads where it is not (8192 x 768 fp32 6 us).
template <class T, int GS>
__global__ __launch_bounds__(256) void quantize(const T* __restrict__ W, u32x4* __restrict__ codes,
                                                __bf16* __restrict__ scales, int64_t N, int K, int KB, int64_t tiles) {
  const int l = threadIdx.x & 63, i = l & 15, h = l >> 4;
  const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;  // wave-uniform
  const int64_t rt = tile / KB;
  const int kb = (int)(tile - rt * KB);
  const int64_t row = rt * kTileRows + i;
  Raw<T> w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = kTileCols * kb + 32 * j + 8 * h;
    w[j].load(W + min(row, N - 1) * K + min(k, K - 8));
    w[j].keep(row < N && k < K);
  }
  unsigned m[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = max_over_h(w[j].most());
  }
  u32x4 out;
  float s[4 / GS];
#pragma unroll
  for (int q = 0; q < 4 / GS; ++q) {
    unsigned g = m[q * GS];
#pragma unroll
    for (int j = 1; j < GS; ++j) g = max(g, m[q * GS + j]);
    const float top = float_of(g);
    const bool fast = top > 0x1p-96f && top < 0x1p96f;
    // top / 6, correctly rounded in the same way
    constexpr float sixth = 1.f / 6.f;
    float ratio = top * sixth;
    ratio = __builtin_fmaf(__builtin_fmaf(-6.f, ratio, top), sixth, ratio);
    if (!fast) ratio = top / 6.f;
    s[q] = g >= 0x7f800000u ? __builtin_nanf("") : pgn_f32(pgn_bf16(ratio));
    float inv = __builtin_amdgcn_rcpf(s[q]);
    inv = __builtin_fmaf(__builtin_fmaf(-s[q], inv, 1.f), inv, inv);
    const auto over = [&](float w) {
      const float t = w * inv;
      return __builtin_fmaf(__builtin_fmaf(-t, s[q], w), inv, t);
    };
#pragma unroll
    for (int j = q * GS; j < (q + 1) * GS; ++j) {
      unsigned a = 0u;
      a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, over(w[j].get(0)), over(w[j].get(1)), 1.f, 0);
      a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, over(w[j].get(2)), over(w[j].get(3)), 1.f, 1);
      a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, over(w[j].get(4)), over(w[j].get(5)), 1.f, 2);
      a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, over(w[j].get(6)), over(w[j].get(7)), 1.f, 3);
      if (!fast) {
        a = 0u;
        if (s[q] > 0.f)  // (zeros and NaN scales: codes 0)
#pragma unroll
          for (int e = 0; e < 8; ++e) a |= exact_code(w[j].get(e), s[q]) << (4 * e);
      }
      out[j] = a;
    }
  }
  codes[tile * 64 + l] = out;
  if (h == 0) {
    __bf16* sp = scales + (tile * kTileRows + i) * (4 / GS);
#pragma unroll
    for (int q = 0; q < 4 / GS; ++q) sp[q] = pgn_bf16(s[q]);
  }
}

// How a wave writes the weights of a tile: 16 bytes to a lane, a row's 128 columns side by side, so that memory is written in
// whole lines (with the lanes of the codes' layout a row's piece is 64 bytes: 32768 x 4096 bf16 in 77 us, so in 67), and past
// the caches where the rows are whole lines (50; rows of 2000 bytes 7.6 instead of 6.8).
template <class T>
struct Rows {
  static constexpr int kCols = 16 / (int)sizeof(T), kLanes = kTileCols / kCols, kAtOnce = 64 / kLanes,
                       kTurns = kTileRows / kAtOnce;
  int row, col;  // of the lane's first vector; the next one's row is kAtOnce further
  PGN_DEVICE explicit Rows(int l) : row(l / kLanes), col(l % kLanes * kCols) {}
  // where codes of these columns lie in the tile: the 32-bit word, and its shift
  PGN_DEVICE int word(int turn) const {
    const int k8 = col >> 3;
    return ((k8 & 3) * 16 + row + kAtOnce * turn) * 4 + (k8 >> 2);
  }
  PGN_DEVICE int shift() const { return (col & 7) * 4; }
};
// One wave a tile, whose four or eight vectors a lane depend on nothing but their own word and scale. LINES: the weight's rows
// are whole lines of 128 bytes. Bound by the bytes written.
template <class T, int GS, bool LINES>
__global__ __launch_bounds__(256) void dequantize(const unsigned* __restrict__ codes, const __bf16* __restrict__ scales,
                                                  T* __restrict__ W, int64_t N, int K, int KB, int64_t tiles) {
  using R = Rows<T>;
  const int l = threadIdx.x & 63;
  const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int64_t rt = tile / KB;
  const int k = kTileCols * (int)(tile - rt * KB);
  const R at(l);
  unsigned c[R::kTurns];
  float s[R::kTurns];
#pragma unroll
  for (int u = 0; u < R::kTurns; ++u) {
    c[u] = codes[tile * 256 + at.word(u)] >> at.shift();
    s[u] = pgn_f32(scales[(tile * kTileRows + at.row + R::kAtOnce * u) * (4 / GS) + at.col / (32 * GS)]);
  }
#pragma unroll
  for (int u = 0; u < R::kTurns; ++u) {
    const int64_t row = rt * kTileRows + at.row + R::kAtOnce * u;
    u32x4 o;
#define PGN_PAIR(P)                                                                                          \
  if constexpr (2 * P < R::kCols) {                                                                          \
    const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, P);                                  \
    if constexpr (R::kCols == 8) {                                                                           \
      const bf16x2 r{pgn_bf16(s[u] * v[0]), pgn_bf16(s[u] * v[1])};                                          \
      o[P] = __builtin_bit_cast(unsigned, r);                                                                \
    } else {                                                                                                 \
      o[2 * P & 3] = bits_of(s[u] * v[0]);                                                                   \
      o[(2 * P + 1) & 3] = bits_of(s[u] * v[1]);                                                             \
    }                                                                                                        \
  }
    PGN_PAIR(0)
    PGN_PAIR(1)
    PGN_PAIR(2)
    PGN_PAIR(3)
#undef PGN_PAIR
    if (row < N && k + at.col < K) {
      u32x4* const to = reinterpret_cast<u32x4*>(W + row * K + k + at.col);
      if constexpr (LINES) __builtin_nontemporal_store(o, to);
      else *to = o;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// rows times a weight

// A word of codes as a matrix operand.
PGN_DEVICE bf16x8 operand(unsigned c) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 1),
               d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, 1.f, 3);
  return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// z in three bf16 parts whose sum it is exactly: each takes the next 8 bits, by truncation. An infinity or NaN is its first
// part alone.
PGN_DEVICE void split8(const float (&z)[8], bf16x8 (&part)[3]) {
  unsigned u[3][8];
  float r[8], any = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    u[0][e] = bits_of(z[e]) & 0xffff0000u;
    r[e] = z[e] - float_of(u[0][e]);
    any += r[e];
  }
  if (any != any) {  // an infinity or NaN less itself is NaN
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned b = bits_of(z[e]);
      if ((b & 0x7f800000u) == 0x7f800000u) {
        u[0][e] |= b & 0x7fffffu ? 0x400000u : 0u;  // (a NaN whose bits are all low stays one)
        r[e] = 0.f;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    u[1][e] = bits_of(r[e]) & 0xffff0000u;
    u[2][e] = bits_of(r[e] - float_of(u[1][e]));
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_amdgcn_perm(u[p][2 * e + 1], u[p][2 * e], 0x07060302u);
    part[p] = __builtin_bit_cast(bf16x8, o);
  }
}

// Sixteen bytes of results.
template <class T>
struct Vec;
template <>
struct Vec<float> {
  f32x4 a;
  PGN_DEVICE void load(const float* p) { a = *reinterpret_cast<const f32x4*>(p); }
  PGN_DEVICE void store(float* p) const { *reinterpret_cast<f32x4*>(p) = a; }
  PGN_DEVICE float get(int e) const { return a[e]; }
  PGN_DEVICE void set(int e, float v) { a[e] = v; }
};
template <>
struct Vec<__bf16> {
  bf16x8 a;
  PGN_DEVICE void load(const __bf16* p) { a = *reinterpret_cast<const bf16x8*>(p); }
  PGN_DEVICE void store(__bf16* p) const { *reinterpret_cast<bf16x8*>(p) = a; }
  PGN_DEVICE float get(int e) const { return (float)a[e]; }
  PGN_DEVICE void set(int e, float v) { a[e] = pgn_bf16(v); }
};

// Mean and 1 / sigma of a row, in all lanes of a wave: the sum, then the squares about the mean. Up to 1024 columns the row
// stays in registers, with its loads issued long before; longer ones are read twice.
template <class T>
struct RowStats {
  static constexpr int H = 2;
  Raw<T> raw[H];
  PGN_DEVICE void load(const T* row, int K, int l, int k0 = 0) {
#pragma unroll
    for (int u = 0; u < H; ++u) raw[u].load(row + min(k0 + 8 * (l + 64 * u), K - 8));
  }
  PGN_DEVICE void get(const T* row, int K, float eps, int l, float& mean, float& rstd) {
    auto total = [&](auto&& f) PGN_INLINE {
      float s = 0.f;
      for (int k0 = 0; k0 < K; k0 += 512 * H) {
        if (K > 512 * H) load(row, K, l, k0);
#pragma unroll
        for (int u = 0; u < H; ++u) {
          float t = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) t += f(raw[u].get(e));
          s += k0 + 8 * (l + 64 * u) < K ? t : 0.f;
        }
      }
      return group_sum<64>(s);
    };
    mean = total([](float v) { return v; }) / (float)K;
    const float m = mean, var = total([m](float v) { return (v - m) * (v - m); }) / (float)K;
    rstd = 1.f / sqrtf(var + eps);
  }
};

// Eight columns of a row as P bf16 parts, normalised with LN; zeros past the last column (tail), where the load was of
// others. (K is a multiple of 8. Loads stand under no condition: behind one the compiler cannot count them, and waits for
// those of the next chunk before it uses this one's. The norm's weights are loaded here: with the row's, they took longer.)
template <class T, int P, bool LN>
PGN_DEVICE void stage8(Raw<T> raw, const T* lnw, const T* lnb, float mean, float rstd, int k, int K, bool tail,
                       bf16x8 (&part)[P]) {
  if (tail) raw.keep(k < K);
  if constexpr (P == 1) {
    part[0] = __builtin_bit_cast(bf16x8, raw.a);
  } else {
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = raw.get(e);
    if constexpr (LN) {
      Raw<T> g, b;
      g.load(lnw + min(k, K - 8));
      b.load((lnb ? lnb : lnw) + min(k, K - 8));
      if (tail) g.keep(k < K);
      b.keep(k < K && lnb);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = (z[e] - mean) * rstd * g.get(e) + b.get(e);
    }
    split8(z, part);
  }
}

// A tile's scales of one row: 4 / GS bf16 numbers in one or two words.
template <int GS>
struct Scales {
  unsigned w[GS == 1 ? 2 : 1];
  PGN_DEVICE void load(const __bf16* p) {
    if constexpr (GS == 1) {
      const i32x2 v = *reinterpret_cast<const i32x2*>(p);
      w[0] = (unsigned)v[0];
      w[1] = (unsigned)v[1];
    } else if constexpr (GS == 2) {
      w[0] = *reinterpret_cast<const unsigned*>(p);
    } else {
      w[0] = *reinterpret_cast<const unsigned short*>(p);
    }
  }
  PGN_DEVICE float get(int q) const {
    const unsigned v = w[GS == 1 ? q >> 1 : 0];
    return q & 1 ? float_of(v & 0xffff0000u) : bf16_bits(v);
  }
};

// acc += one block of 128 columns: RT x NT tiles. x(p, r, ks) is the rows' operand, c and s the tiles' codes and scales.
template <int P, int GS, int RT, int NT, class X>
PGN_DEVICE void block(f32x4 (&acc)[RT][NT], const u32x4 (&c)[NT], const Scales<GS> (&s)[NT], X&& x) {
  constexpr int G = 4 / GS;
  const f32x4 zero{0.f, 0.f, 0.f, 0.f};
  if constexpr (RT * NT < 4) {
    // few tiles: every group's and part's sum a chain of its own, so that the products need not wait for each other
    f32x4 d[G][P][RT][NT];
#pragma unroll
    for (int g = 0; g < GS; ++g)
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const int ks = q * GS + g;
        bf16x8 b[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) b[t] = operand(c[t][ks]);
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const bf16x8 a = x(p, r, ks);
#pragma unroll
            for (int t = 0; t < NT; ++t) d[q][p][r][t] = pgn_mfma(a, b[t], g ? d[q][p][r][t] : zero);
          }
      }
#pragma unroll
    for (int q = 0; q < G; ++q)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          f32x4 v = d[q][P - 1][r][t];  // the smallest parts first
#pragma unroll
          for (int p = P - 2; p >= 0; --p) v += d[q][p][r][t];
          acc[r][t] += s[t].get(q) * v;
        }
  } else if constexpr (P == 1 && RT * NT >= 16) {
    // many tiles: a group's operands of the rows are kept, the tiles of columns taken one after the other (all at once, the
    // sums leave no registers)
#pragma unroll
    for (int q = 0; q < G; ++q) {
      bf16x8 a[GS][RT];
#pragma unroll
      for (int g = 0; g < GS; ++g)
#pragma unroll
        for (int r = 0; r < RT; ++r) a[g][r] = x(0, r, q * GS + g);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 d[RT];
#pragma unroll
        for (int g = 0; g < GS; ++g) {
          const bf16x8 b = operand(c[t][q * GS + g]);
#pragma unroll
          for (int r = 0; r < RT; ++r) d[r] = pgn_mfma(a[g][r], b, g ? d[r] : zero);
        }
        const float v = s[t].get(q);
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r][t] += v * d[r];
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < G; ++q) {
      f32x4 d[RT][NT];
#pragma unroll
      for (int g = 0; g < GS; ++g) {
        const int ks = q * GS + g;
        bf16x8 b[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) b[t] = operand(c[t][ks]);
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const bf16x8 a = x(p, r, ks);
#pragma unroll
            for (int t = 0; t < NT; ++t) d[r][t] = pgn_mfma(a, b[t], g || p < P - 1 ? d[r][t] : zero);
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float v = s[t].get(q);
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r][t] += v * d[r][t];
      }
    }
  }
}

template <class T>
PGN_DEVICE void finish(float v, int row, int col, int N, const T* bias, int act, const T* resid, T* y) {
  if (bias) v += (float)bias[col];
  if (act == 1) v = pgn_gelu_erf(v);
  const size_t off = (size_t)row * N + col;
  if (resid) v += (float)resid[off];
  y[off] = (T)v;
}

// The same of one result to a thread, its bias and residual loaded as the kernel starts (of x where there is none).
template <class T>
struct Epilogue {
  T bias, resid;
  PGN_DEVICE void load(const T* x, const T* bp, const T* rp, int row, int col, int n, int N) {
    bias = *(bp ? bp + min(col, N - 1) : x);
    resid = *(rp ? rp + (size_t)min(row, n - 1) * N + min(col, N - 1) : x);
  }
  PGN_DEVICE void finish(float v, int row, int col, int N, const T* bp, int act, const T* rp, T* y) const {
    v += bp ? (float)bias : 0.f;
    if (act == 1) v = pgn_gelu_erf(v);
    v += rp ? (float)resid : 0.f;
    y[(size_t)row * N + col] = (T)v;
  }
};

// Sixteen rows are staged in whole lines: sixteen lanes take 128 neighbouring columns of a row (four lanes 32 of each row: up
// to 1.7 times as long, 16 x 4096 x 14336 bf16 16.1 us against 9.3). Their pieces are written a pitch apart and read a row
// apart, so a pitch of one piece past 16 keeps both off each other's banks.
constexpr int kPitch = 17;

// MR = 1, 4 or 16 rows and one tile of 16 columns to a workgroup, its WK waves sharing the blocks of 128 contracted columns.
// A wave stages its own columns of the rows in LDS of its own, so that only the sums' joining needs a barrier (and the
// norms of several rows another). A wave's loads of CBW blocks are issued at once; while it waits for the next, others of the
// compute unit work (their loads issued ahead, in registers of their own: 64 x 704 x 2816 7.8 -> 9.0 us). One row of 16384 x
// 4096 in groups of 32 takes 7.8 us, 4.8 TB/s of codes and scales, and is bound by them; small products by the chain of a launch,
// the row's moments, one round of loads and the join (1 x 2328 x 768 with a norm 3.7 us).
template <class T, int P, bool LN, int GS, int MR, int WK, int CBW>
__global__ __launch_bounds__(64 * WK) void few(const T* __restrict__ x, const u32x4* __restrict__ codes,
                                               const __bf16* __restrict__ scales, const T* __restrict__ lnw,
                                               const T* __restrict__ lnb, float eps, const T* __restrict__ bias, int act,
                                               const T* resid, T* y, int n, int N, int K, int KB, int ctiles,
                                               int rblocks) {
  constexpr int U = CBW * MR / 4;  // pieces of 8 columns a lane stages
  constexpr int S = MR == 16 ? kPitch : MR;
  static_assert(CBW * MR % 4 == 0 && (MR == 1 || MR == 4 || MR == 16) && 16 * MR <= 64 * WK, "");
  extern __shared__ __align__(16) char smem[];
  __shared__ float sums[WK][MR][16];
  __shared__ float stat[MR][2];
  const int tid = threadIdx.x, l = tid & 63, wk = __builtin_amdgcn_readfirstlane(tid >> 6), i = l & 15, h = l >> 4;
  // workgroups of the same columns run on one XCD (their numbers differ by multiples of 8)
  int ct = blockIdx.x, rb = 0;
  if (rblocks > 1) {
    const int rest = blockIdx.x >> 3;
    rb = rest % rblocks;
    ct = rest / rblocks * 8 + (blockIdx.x & 7);
  }
  if (ct >= ctiles) return;
  bf16x8* const mine = reinterpret_cast<bf16x8*>(smem) + wk * P * CBW * 16 * S;  // [P][CBW * 16][S]
  const int row0 = rb * MR;
  const int row = row0 + (tid >> 4), col = ct * 16 + (tid & 15);  // the result this thread ends with
  // piece u of this lane: 8 columns k8 of the wave's blocks, all its blocks' pieces in a row, of row m
  auto k8 = [&](int u) { return MR == 16 ? 16 * (u / 4) + i : u * (64 / MR) + l / MR; };
  auto m = [&](int u) { return MR == 16 ? 4 * (u % 4) + h : l % MR; };
  const T* const xb = x + (size_t)row0 * K;
  constexpr int R = MR == 16 ? 4 : 1;  // rows that a lane stages pieces of
  unsigned xr[R];
#pragma unroll
  for (int u = 0; u < R; ++u) xr[u] = (unsigned)(min(m(u), n - 1 - row0) * K);
  auto column = [&](int kb0, int u) { return kTileCols * (kb0 + WK * (k8(u) >> 4)) + 8 * (k8(u) & 15); };
  constexpr int kRows = LN ? (MR + WK - 1) / WK : 1;  // rows whose moments a wave forms (all form the one of MR = 1)
  RowStats<T> stats[kRows];
  auto stat_row = [&](int r) { return x + (size_t)min(row0 + (MR == 1 ? 0 : (wk + WK * r) % MR), n - 1) * K; };
  Raw<T> raw[U];
  u32x4 c[CBW][1];
  Scales<GS> s[CBW][1];
  auto load = [&](int kb0) PGN_INLINE {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].load(xb + (xr[u % R] + (unsigned)min(column(kb0, u), K - 8)));
#pragma unroll
    for (int j = 0; j < CBW; ++j) {
      const size_t tile = (size_t)ct * KB + min(kb0 + WK * j, KB - 1);  // (past the last: not used)
      c[j][0] = codes[tile * 64 + l];
      s[j][0].load(scales + (tile * 16 + i) * (4 / GS));
    }
  };
  if constexpr (LN)
#pragma unroll
    for (int r = 0; r < kRows; ++r) stats[r].load(stat_row(r), K, l);
  load(wk);
  Epilogue<T> end;
  if (wk < (16 * MR + 63) / 64) end.load(x, bias, resid, row, col, n, N);
  float mean[R], rstd[R];
  if constexpr (LN) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      stats[r].get(stat_row(r), K, eps, l, mean[0], rstd[0]);
      if (MR > 1 && l == 0 && wk + WK * r < MR) {
        stat[wk + WK * r][0] = mean[0];
        stat[wk + WK * r][1] = rstd[0];
      }
    }
    if constexpr (MR > 1) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < R; ++u) {
        mean[u] = stat[m(u)][0];
        rstd[u] = stat[m(u)][1];
      }
    }
  }
  f32x4 acc[1][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}};
  for (int kb0 = wk; kb0 < KB; kb0 += WK * CBW) {
    if (kb0 != wk) load(kb0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (past the last block; the lanes of one row's pieces have different ones)
      if (MR > 1 && kb0 + WK * (MR == 16 ? u / 4 : u * (64 / MR) / 16) >= KB) break;
      bf16x8 part[P];
      stage8<T, P, LN>(raw[u], lnw, lnb, LN ? mean[u % R] : 0.f, LN ? rstd[u % R] : 1.f, column(kb0, u), K,
                       K % kTileCols != 0, part);
#pragma unroll
      for (int p = 0; p < P; ++p) mine[(p * CBW * 16 + k8(u)) * S + m(u)] = part[p];
    }
    // the wave reads what its own lanes wrote: LDS works in a wave's order, the compiler is kept to it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < CBW; ++j)
      if (kb0 + WK * j < KB)
        block<P, GS>(acc, c[j], s[j],
                     [&](int p, int, int ks) { return mine[(p * CBW * 16 + j * 16 + 4 * ks + h) * S + i % MR]; });
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  if (h < (MR + 3) / 4)
#pragma unroll
    for (int r = 0; r < (MR < 4 ? MR : 4); ++r) sums[wk][4 * h + r][i] = acc[0][0][r];
  __syncthreads();
  if (tid < 16 * MR && row < n && col < N) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < WK; ++k) v += sums[k][tid >> 4][tid & 15];
    end.finish(v, row, col, N, bias, act, resid, y);
  }
}

// Waves to a SIMD: two workgroups of eight share a compute unit, but for those whose LDS leaves room for one (64 rows; two
// blocks of three parts) and those of several parts in groups of 32, whose scales and sums would spill (fp32 512 x 16384 x 1024
// 70.8 us with two, 58.8 with one).
template <int P, int GS, int kWaves, int RT, int U>
constexpr int waves_per_simd() {
  return RT == 4 || (kWaves == 8 && P > 1 && (P * U > 4 || GS == 1)) ? 2 : 4;
}

// More rows. A workgroup's share: 16 RT rows, WN NT tiles of 16 columns, WK waves sharing the contracted columns of each (WN
// WK waves). Rows go to LDS in P bf16 parts, a chunk of CB blocks of 128 columns at a time, as the matrix core takes them;
// codes straight to registers. A chunk's loads are under way while the one before it is multiplied. Large products are bound by
// instructions and by waits: beside a matrix instruction of 16 cycles stand its share of the conversions (4 / RT) and of the
// scaling of its sums (2 in groups of 64), and two vector instructions beside one cost 2 cycles, a third 4 more; and two waves a
// SIMD that meet at a chunk's barrier do not fill each other's waits. 512 x 8192 x 4096 bf16: 36.5 us, 945 TFLOP/s, the matrix
// cores busy 41% of the time, a wave waiting 30% of it; fp32 rows and normalised ones are three such products (512 x 16384 x
// 1024 48 us).
template <class T, int P, bool LN, int GS, int kWaves, int RT, int U, int WK, int NT>
__global__ __launch_bounds__(64 * kWaves, (waves_per_simd<P, GS, kWaves, RT, U>())) void linear(
    const T* __restrict__ x, const u32x4* __restrict__ codes, const __bf16* __restrict__ scales, const T* __restrict__ lnw,
    const T* __restrict__ lnb, float eps, const T* __restrict__ bias, int act, const T* resid, T* y, int n, int N, int K,
    int KB, int ctiles, int rblocks) {
  // a wave's loads of 4 rows by 128 columns: U in a chunk, of 16 rows' quarters and blocks in turn, so of R row tiles
  constexpr int WN = kWaves / WK, CB = U * kWaves / (4 * RT), CK8 = 16 * CB, CBW = CB / WK;
  constexpr int R = 4 * RT > kWaves ? 4 * RT / kWaves : 1, step = CK8 / (U / R);
  static_assert(CBW * WK * 4 * RT == U * kWaves && U % R == 0 && kWaves % 4 == 0, "");
  extern __shared__ __align__(16) char smem[];
  __shared__ float stat[2][16 * RT];
  bf16x8* const buf = reinterpret_cast<bf16x8*>(smem);  // [2 chunks][P][RT][CK8][kPitch]
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = l & 15, h = l >> 4, wk = w % WK, wn = w / WK;
  // workgroups of the same columns run on one XCD (their numbers differ by multiples of 8)
  int cg = blockIdx.x, rb = 0;
  if (rblocks > 1) {
    const int rest = blockIdx.x >> 3;
    rb = rest % rblocks;
    cg = rest / rblocks * 8 + (blockIdx.x & 7);
  }
  const int ct0 = cg * WN * NT + wn * NT, row0 = rb * 16 * RT;
  if (cg * WN * NT >= ctiles) return;
  const int nch = (KB + CB - 1) / CB;

  // staging: this thread's row, and its first 8-column piece of a chunk. Addresses are a wave's own part plus a lane's 32
  // bits that no chunk changes: the vector unit has no arithmetic to spare (below).
  const int sm = w % 4 * 4 + h, sk = w / (4 * RT) * 16 + i;
  auto srt = [&](int u) { return (w / 4 + u % R * (kWaves / 4)) % RT; };
  const T* const xb = x + (size_t)row0 * K;
  unsigned xrow[R];
#pragma unroll
  for (int r = 0; r < R; ++r) xrow[r] = (unsigned)(min(16 * srt(r) + sm, n - 1 - row0) * K);
  const int full = K / (8 * CK8);  // chunks that lie in the row whole
  Raw<T> raw[U];
  auto load_x = [&](int c) PGN_INLINE {
    if (c < full) {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u].load(xb + (size_t)(8 * (c * CK8 + u / R * step)) + (xrow[u % R] + 8 * sk));
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u].load(xb + (xrow[u % R] + (unsigned)min(8 * (c * CK8 + sk + u / R * step), K - 8)));
    }
  };
  u32x4 cw[CBW][NT], cn[CBW][NT];  // this chunk's codes, the next one's
  Scales<GS> sw[CBW][NT], sn[CBW][NT];
  auto load_w = [&](int c, u32x4 (&cc)[CBW][NT], Scales<GS> (&ss)[CBW][NT]) PGN_INLINE {
#pragma unroll
    for (int j = 0; j < CBW; ++j)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const size_t tile = (size_t)min(ct0 + t, ctiles - 1) * KB + min(c * CB + wk + WK * j, KB - 1);
        cc[j][t] = (codes + tile * 64)[(unsigned)l];
        ss[j][t].load(scales + tile * (16 * 4 / GS) + (unsigned)(i * (4 / GS)));
      }
  };
  // one result to a thread in the smallest tiles, whose latency counts
  constexpr int C = WN * NT * 16, all = 16 * RT * C / (64 * kWaves), most = 16 / (int)sizeof(T),
                V = all < 1 ? 1 : all < most ? all : most;
  constexpr bool single = V == 1 && 16 * RT * C == 64 * kWaves;
  constexpr int kRows = LN ? 16 * RT / kWaves : 1;  // rows whose moments a wave forms
  RowStats<T> stats[kRows];
  auto stat_row = [&](int r) { return x + (size_t)min(row0 + w + kWaves * r, n - 1) * K; };
  if constexpr (LN)
#pragma unroll
    for (int r = 0; r < kRows; ++r) stats[r].load(stat_row(r), K, l);
  load_x(0);
  load_w(0, cw, sw);
  Epilogue<T> end;
  if constexpr (single) end.load(x, bias, resid, row0 + tid / C, cg * C + tid % C, n, N);
  float mean[R], rstd[R];
  if constexpr (LN) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      stats[r].get(stat_row(r), K, eps, l, mean[0], rstd[0]);
      if (l == 0) {
        stat[0][w + kWaves * r] = mean[0];
        stat[1][w + kWaves * r] = rstd[0];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = stat[0][16 * srt(r) + sm];
      rstd[r] = stat[1][16 * srt(r) + sm];
    }
  }
  auto store_x = [&](int c) PGN_INLINE {
    bf16x8* const to = buf + (c & 1) * P * RT * CK8 * kPitch;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k8 = sk + u / R * step;
      bf16x8 part[P];
      stage8<T, P, LN>(raw[u], lnw, lnb, LN ? mean[u % R] : 0.f, LN ? rstd[u % R] : 1.f, 8 * (c * CK8 + k8), K, c >= full, part);
#pragma unroll
      for (int p = 0; p < P; ++p) to[((p * RT + srt(u)) * CK8 + k8) * kPitch + sm] = part[p];
    }
  };
  store_x(0);

  f32x4 acc[RT][NT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int c, const u32x4 (&cc)[CBW][NT], const Scales<GS> (&ss)[CBW][NT]) PGN_INLINE {
    const bf16x8* const from = buf + (c & 1) * P * RT * CK8 * kPitch;
#pragma unroll
    for (int j = 0; j < CBW; ++j) {
      if (c * CB + wk + WK * j < KB) {
        const bf16x8* const at = from + ((wk + WK * j) * 16 + h) * kPitch + i;
        block<P, GS>(acc, cc[j], ss[j], [&](int p, int r, int ks) { return at[((p * RT + r) * CK8 + 4 * ks) * kPitch]; });
      }
    }
  };
  // (two chunks a turn, so that codes need not be moved from one set of registers to the other)
  auto turn = [&](int c, u32x4 (&c0)[CBW][NT], Scales<GS> (&s0)[CBW][NT], u32x4 (&c1)[CBW][NT],
                  Scales<GS> (&s1)[CBW][NT]) PGN_INLINE {
    __syncthreads();
    load_x(c + 1);
    load_w(c + 1, c1, s1);
    multiply(c, c0, s0);
    store_x(c + 1);
  };
  int c = 0;
  for (; c + 2 < nch; c += 2) {
    turn(c, cw, sw, cn, sn);
    turn(c + 1, cn, sn, cw, sw);
  }
  if (c + 1 < nch) {
    turn(c, cw, sw, cn, sn);
    __syncthreads();
    multiply(c + 1, cn, sn);
  } else {
    __syncthreads();
    multiply(c, cw, sw);
  }

  // The sums go through LDS, wave wk's at [wk][row][column], and V consecutive columns of a row to a thread: the waves' shares
  // are added in order, and rows are read and written in whole vectors. (A pitch of 4 past 16: a store's four rows of 16
  // columns fall on different banks.)
  constexpr int S = C + 4;
  float* const part = reinterpret_cast<float*>(smem);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[(wk * 16 * RT + 16 * r + 4 * h + e) * S + (wn * NT + t) * 16 + i] = acc[r][t][e];
  __syncthreads();
  const bool whole = N % most == 0;  // every vector lies in a row and at a vector's address
  for (int o = tid; o < 16 * RT * C / V; o += 64 * kWaves) {
    const int r = o / (C / V), c = o % (C / V) * V, row = row0 + r, col = cg * C + c;
    if (row >= n || col >= N) continue;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = part[r * S + c + e];
#pragma unroll
    for (int k = 1; k < WK; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += part[(k * 16 * RT + r) * S + c + e];
    const size_t off = (size_t)row * N + col;
    if constexpr (single) {
      end.finish(v[0], row, col, N, bias, act, resid, y);
    } else if (V == most && whole) {
      Vec<T> q;
      if (bias) {
        q.load(bias + col);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += q.get(e);
      }
      if (act == 1)
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = pgn_gelu_erf(v[e]);
      if (resid) {
        q.load(resid + off);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += q.get(e);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) q.set(e, v[e]);
      q.store(y + off);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (col + e < N) finish(v[e], row, col + e, N, bias, act, resid, y);
    }
  }
}

constexpr size_t kPlainLds = 60 << 10;  // LDS that a launch may ask for without raising the limit, statistics apart

struct Call {
  const void *x, *codes, *scales, *lnw, *lnb, *bias, *resid;
  void* y;
  float eps;
  int act, n, N, K;
  hipStream_t st;
};

template <class T, int P, bool LN, int GS, int MR, int WK, int CBW>
int launch_few(const Call& a) {
  const int KB = (a.K + kTileCols - 1) / kTileCols, ctiles = (a.N + 15) / 16, rblocks = (a.n + MR - 1) / MR;
  const int64_t blocks = rblocks > 1 ? (int64_t)(ctiles + 7) / 8 * 8 * rblocks : ctiles;
  constexpr size_t lds = (size_t)WK * P * CBW * 16 * (MR == 16 ? kPitch : MR) * 16, sums = (size_t)WK * MR * 16 * 4;
  static_assert(lds + sums <= 159 << 10, "");
  const auto fn = few<T, P, LN, GS, MR, WK, CBW>;
  if constexpr (lds + sums > kPlainLds) {
    const hipError_t e = pgn_lds_limit(reinterpret_cast<const void*>(fn), lds);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(64 * WK), lds, a.st, (const T*)a.x, (const u32x4*)a.codes,
                     (const __bf16*)a.scales, (const T*)a.lnw, (const T*)a.lnb, a.eps, (const T*)a.bias, a.act,
                     (const T*)a.resid, (T*)a.y, a.n, a.N, a.K, KB, ctiles, rblocks);
  PGN_RETURN_LAUNCH();
}

template <class T, int P, bool LN, int GS, int kWaves, int RT, int U, int WK, int NT>
int launch(const Call& a) {
  constexpr int CB = U * kWaves / (4 * RT), WN = kWaves / WK;
  const int KB = (a.K + kTileCols - 1) / kTileCols, ctiles = (a.N + 15) / 16;
  const int rblocks = (a.n + 16 * RT - 1) / (16 * RT), groups = (ctiles + WN * NT - 1) / (WN * NT);
  const int64_t blocks = rblocks > 1 ? (int64_t)(groups + 7) / 8 * 8 * rblocks : groups;
  constexpr size_t chunk = (size_t)P * U * kWaves * 64 * kPitch, join = (size_t)WK * 16 * RT * (WN * NT * 16 + 4) * 4;
  const size_t lds = std::max(KB > CB ? 2 * chunk : chunk, join);
  const auto fn = linear<T, P, LN, GS, kWaves, RT, U, WK, NT>;
  static_assert(std::max(2 * chunk, join) <= 159 << 10, "");
  if (lds > kPlainLds) {
    const hipError_t e = pgn_lds_limit(reinterpret_cast<const void*>(fn), std::max(2 * chunk, join));
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(64 * kWaves), lds, a.st, (const T*)a.x, (const u32x4*)a.codes,
                     (const __bf16*)a.scales, (const T*)a.lnw, (const T*)a.lnb, a.eps, (const T*)a.bias, a.act,
                     (const T*)a.resid, (T*)a.y, a.n, a.N, a.K, KB, ctiles, rblocks);
  PGN_RETURN_LAUNCH();
}

// Rows and columns of a workgroup, measured in us. Up to four rows a workgroup is one tile of columns. Beyond, the
// smallest tile of rows by columns that leaves no compute unit a second workgroup, as each stages its rows itself and a
// short row's cost is its chain of barriers. 16 x 16, no barrier between blocks, while there are 256 of those or fewer
// (fp32, against 16 x 64: 16 x 768 x 768 3.5 and 4.1, 16 x 2328 x 768 with a norm 5.8 and 6.5; 512 of them, bf16, 6.7
// and 6.2), with sixteen waves where there is one part, which leaves its loads the time (16 x 4096 x 14336 bf16 9.3,
// with eight 11.0). Then 16 x 64, 32 x 128 and 32 x 256 (fp32: 16 x 2328 x 768 5.7, 8.4, 10.7; 128 x 2328 x 768 10.1,
// 9.3, 11.5; 512 x 2328 x 768 23.8, 17.2, 13.0). 32 x 128 has sixteen waves, but eight with two tiles of columns each
// where three parts make reading the rows the limit and no norm needs the waves (64 x 8192 x 768 8.2, with sixteen 8.8;
// with a norm 12.3 and 11.8) or groups of 32 the registers (8.4 and 13.4). 32 x 256 has sixteen waves for one round of
// workgroups, eight for more, two workgroups to a compute unit (512 x 16384 x 1024 bf16 23.7, with sixteen 27.7; fp32
// 48 and 51, 511 x 16880 x 256 18.3 and 24.8; one round, 512 x 2328 x 768, 17.1 and 14.3). One part's eight waves take
// 64 x 256, half the conversions and reads of rows, where the contracted axis is long and workgroups of one to a
// compute unit fill the last round or nearly: 512 x 8192 x 4096 36.4 against 39.4 with 32 x 256, in groups of 32 41.9
// against 45.6, 2048 deep 20.4 against 21.4; with the last round a quarter full, 640 x 8192 x 4096 67 against 55.
template <class T, int P, bool LN, int GS>
int by_rows(const Call& a) {
  if (a.n == 1) return launch_few<T, P, LN, GS, 1, 8, 4>(a);
  if (a.n <= 4) return launch_few<T, P, LN, GS, 4, 8, 2>(a);
  const auto blocks = [&](int64_t rows, int64_t cols) { return (a.n + rows - 1) / rows * ((a.N + cols - 1) / cols); };
  if (blocks(16, 16) <= 256) return launch_few<T, P, LN, GS, 16, P == 1 ? 16 : 8, 1>(a);
  if (blocks(16, 64) <= 256) return launch<T, P, LN, GS, 16, 1, 1, 4, 1>(a);
  if (blocks(32, 128) <= 256) {
    if constexpr (P == 3 && (!LN || GS == 1)) return launch<T, P, LN, GS, 8, 2, 2, 2, 2>(a);
    else return launch<T, P, LN, GS, 16, 2, 1, 2, 1>(a);
  }
  if (blocks(32, 256) > 256) {
    if constexpr (P == 1)
      if (a.K >= 2048 && (a.n + 31) / 32 % 2 == 0 && (blocks(64, 256) + 255) % 256 >= 224)
        return launch<T, P, LN, GS, 8, 4, 4, 2, 4>(a);
    return launch<T, P, LN, GS, 8, 2, P == 1 ? 2 : 1, 1, 2>(a);
  }
  return launch<T, P, LN, GS, 16, 2, 1, 2, 2>(a);
}

template <class T, int P, bool LN>
int by_group(const Call& a, int64_t group) {
  return group == 32 ? by_rows<T, P, LN, 1>(a) : group == 64 ? by_rows<T, P, LN, 2>(a) : by_rows<T, P, LN, 4>(a);
}

bool weight_ok(int64_t N, int64_t K, int64_t group) {
  return N > 0 && N <= ((int64_t)1 << 26) && K > 0 && K <= 65536 && K % 8 == 0 &&
         (group == 32 || group == 64 || group == 128);
}
int64_t tiles_of(int64_t N, int64_t K) {
  return (N + kTileRows - 1) / kTileRows * ((K + kTileCols - 1) / kTileCols);
}
bool aligned(const void* a, const void* b, const void* c) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0;
}

}  // namespace

extern "C" int pragnosia_gen_abi_version(void) { return 1; }

extern "C" int64_t pragnosia_fp4_code_bytes(int64_t N, int64_t K) {
  return weight_ok(N, K, 32) ? tiles_of(N, K) * kTileBytes : PRAGNOSIA_ERR_INVALID_ARGUMENT;
}

extern "C" int64_t pragnosia_fp4_scale_bytes(int64_t N, int64_t K, int64_t group) {
  return weight_ok(N, K, group) ? tiles_of(N, K) * kTileRows * (kTileCols / group) * 2 : PRAGNOSIA_ERR_INVALID_ARGUMENT;
}

namespace {

template <class T, int GS>
void launch_quantize(const void* W, void* codes, void* scales, int64_t N, int K, int64_t tiles, hipStream_t st) {
  hipLaunchKernelGGL((quantize<T, GS>), dim3((unsigned)((tiles + 3) / 4)), dim3(256), 0, st, (const T*)W, (u32x4*)codes,
                     (__bf16*)scales, N, K, (K + kTileCols - 1) / kTileCols, tiles);
}

template <class T, int GS>
void launch_dequantize(const void* codes, const void* scales, void* W, int64_t N, int K, int64_t tiles, hipStream_t st) {
  const auto fn = K % (128 / (int)sizeof(T)) == 0 ? dequantize<T, GS, true> : dequantize<T, GS, false>;
  hipLaunchKernelGGL(fn, dim3((unsigned)((tiles + 3) / 4)), dim3(256), 0, st, (const unsigned*)codes,
                     (const __bf16*)scales, (T*)W, N, K, (K + kTileCols - 1) / kTileCols, tiles);
}

}  // namespace

#define PGN_BY_TYPE(FN, ...)                                     \
  if (bf16) {                                                    \
    if (group == 32) FN<__bf16, 1>(__VA_ARGS__);                 \
    else if (group == 64) FN<__bf16, 2>(__VA_ARGS__);            \
    else FN<__bf16, 4>(__VA_ARGS__);                             \
  } else {                                                       \
    if (group == 32) FN<float, 1>(__VA_ARGS__);                  \
    else if (group == 64) FN<float, 2>(__VA_ARGS__);             \
    else FN<float, 4>(__VA_ARGS__);                              \
  }

extern "C" int pragnosia_fp4_quantize(const void* W, int bf16, void* codes, void* scales, int64_t N, int64_t K,
                                      int64_t group, void* stream) {
  PGN_CHECK_ARG(W && codes && scales && weight_ok(N, K, group) && aligned(W, codes, scales));
  PGN_BY_TYPE(launch_quantize, W, codes, scales, N, (int)K, tiles_of(N, K), (hipStream_t)stream)
  PGN_RETURN_LAUNCH();
}

extern "C" int pragnosia_fp4_dequantize(const void* codes, const void* scales, void* W, int bf16, int64_t N, int64_t K,
                                        int64_t group, void* stream) {
  PGN_CHECK_ARG(W && codes && scales && weight_ok(N, K, group) && aligned(W, codes, scales));
  PGN_BY_TYPE(launch_dequantize, codes, scales, W, N, (int)K, tiles_of(N, K), (hipStream_t)stream)
  PGN_RETURN_LAUNCH();
}

extern "C" int pragnosia_fp4_linear(const void* x, int bf16, const void* codes, const void* scales,
                                    const void* ln_weight, const void* ln_bias, float ln_eps, const void* bias, int act,
                                    const void* resid, void* y, int64_t n, int64_t N, int64_t K, int64_t group,
                                    void* stream) {
  PGN_CHECK_ARG(n >= 0 && n <= ((int64_t)1 << 24) && weight_ok(N, K, group) && (act == 0 || act == 1));
  PGN_CHECK_ARG(n * N < ((int64_t)1 << 31) && n * K < ((int64_t)1 << 31));
  if (n == 0) return PRAGNOSIA_OK;
  PGN_CHECK_ARG(x && codes && scales && y && aligned(x, codes, scales) && aligned(ln_weight, ln_bias, nullptr));
  PGN_CHECK_ARG((ln_weight || !ln_bias) && (!ln_weight || ln_eps >= 0.f));
  const uintptr_t size = bf16 ? 2 : 4, xa = (uintptr_t)x, ya = (uintptr_t)y;
  PGN_CHECK_ARG(aligned(y, bias, resid));
  PGN_CHECK_ARG(xa + (uintptr_t)(n * K) * size <= ya || ya + (uintptr_t)(n * N) * size <= xa);
  const Call a{x, codes, scales, ln_weight, ln_bias, bias, resid, y, ln_eps, act, (int)n, (int)N, (int)K,
               (hipStream_t)stream};
  if (!bf16) return ln_weight ? by_group<float, 3, true>(a, group) : by_group<float, 3, false>(a, group);
  return ln_weight ? by_group<__bf16, 3, true>(a, group) : by_group<__bf16, 1, false>(a, group);
}
