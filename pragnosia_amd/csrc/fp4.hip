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
  PGN_DEVICE void zero() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
  PGN_DEVICE float get(int e) const { return e < 4 ? a[e & 3] : b[e & 3]; }
};
template <>
struct Raw<__bf16> {
  u32x4 a;
  PGN_DEVICE void load(const __bf16* p) { a = *reinterpret_cast<const u32x4*>(p); }
  PGN_DEVICE void zero() { a = u32x4{0u, 0u, 0u, 0u}; }
  PGN_DEVICE float get(int e) const { return e & 1 ? float_of(a[e >> 1] & 0xffff0000u) : bf16_bits(a[e >> 1]); }
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

// One wave a tile. The codes come from the hardware's conversion of w / s, with the quotient a little too large and a
// little too small: where both give the same eight codes no border lies within the quotient's error, elsewhere (about
// one lane in 10^4, and every exact tie) exact_code decides.
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
    if (row < N && k < K) w[j].load(W + row * K + k);
    else w[j].zero();
  }
  unsigned m[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) m[j] = max(m[j], bits_of(w[j].get(e)) & 0x7fffffffu);
    m[j] = max_over_h(m[j]);
  }
  u32x4 out;
  float s[4 / GS];
#pragma unroll
  for (int q = 0; q < 4 / GS; ++q) {
    unsigned g = m[q * GS];
#pragma unroll
    for (int j = 1; j < GS; ++j) g = max(g, m[q * GS + j]);
    s[q] = g >= 0x7f800000u ? __builtin_nanf("") : pgn_f32(pgn_bf16(float_of(g) / 6.f));
    const bool fast = s[q] > 0x1p-100f && s[q] < 0x1p100f;
    const float inv = __builtin_amdgcn_rcpf(s[q]), hi = inv * (1.f + 0x1p-20f), lo = inv * (1.f - 0x1p-20f);
#pragma unroll
    for (int j = q * GS; j < (q + 1) * GS; ++j) {
      unsigned a = 0u, b = 0u;
#define PGN_PAIR(P)                                                                                              \
  a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, w[j].get(2 * P) * hi, w[j].get(2 * P + 1) * hi, 1.f, P);       \
  b = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(b, w[j].get(2 * P) * lo, w[j].get(2 * P + 1) * lo, 1.f, P);
      PGN_PAIR(0)
      PGN_PAIR(1)
      PGN_PAIR(2)
      PGN_PAIR(3)
#undef PGN_PAIR
      if (!(fast && a == b)) {
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

// The eight values of a word of codes, times s.
PGN_DEVICE void decode8(unsigned c, float s, float (&v)[8]) {
#define PGN_PAIR(P)                                                              \
  {                                                                              \
    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, P);         \
    v[2 * P] = s * p[0];                                                         \
    v[2 * P + 1] = s * p[1];                                                     \
  }
  PGN_PAIR(0)
  PGN_PAIR(1)
  PGN_PAIR(2)
  PGN_PAIR(3)
#undef PGN_PAIR
}

PGN_DEVICE void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
  reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
}
PGN_DEVICE void store8(__bf16* p, const float (&v)[8]) {
  bf16x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = pgn_bf16(v[e]);
  *reinterpret_cast<bf16x8*>(p) = o;
}

// One wave a tile.
template <class T, int GS>
__global__ __launch_bounds__(256) void dequantize(const u32x4* __restrict__ codes, const __bf16* __restrict__ scales,
                                                  T* __restrict__ W, int64_t N, int K, int KB, int64_t tiles) {
  const int l = threadIdx.x & 63, i = l & 15, h = l >> 4;
  const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int64_t rt = tile / KB;
  const int kb = (int)(tile - rt * KB);
  const int64_t row = rt * kTileRows + i;
  const u32x4 c = codes[tile * 64 + l];
  const __bf16* sp = scales + (tile * kTileRows + i) * (4 / GS);
  float s[4 / GS];
#pragma unroll
  for (int q = 0; q < 4 / GS; ++q) s[q] = pgn_f32(sp[q]);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = kTileCols * kb + 32 * j + 8 * h;
    float v[8];
    decode8(c[j], s[j / GS], v);
    if (row < N && k < K) store8(W + row * K + k, v);
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

// z in P bf16 parts whose sum it is: exactly with three (each takes the next 8 bits, by truncation), to 16 bits with two,
// rounded with one. An infinity or NaN is its first part alone.
template <int P>
PGN_DEVICE void split8(const float (&z)[8], bf16x8 (&part)[P]) {
  if constexpr (P == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) part[0][e] = pgn_bf16(z[e]);
  } else {
    unsigned u[P][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned b = bits_of(z[e]);
      const bool odd = (b & 0x7f800000u) == 0x7f800000u;
      u[0][e] = (b & 0xffff0000u) | (odd && (b & 0x7fffffu) ? 0x400000u : 0u);  // (a NaN whose bits are all low stays one)
      float r = odd ? 0.f : z[e] - float_of(b & 0xffff0000u);
      if constexpr (P == 3) {
        u[1][e] = bits_of(r) & 0xffff0000u;
        r -= float_of(u[1][e]);
        u[2][e] = bits_of(r);
      } else {
        u[1][e] = bits_of(r);
      }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_amdgcn_perm(u[p][2 * e + 1], u[p][2 * e], 0x07060302u);
      part[p] = __builtin_bit_cast(bf16x8, o);
    }
  }
}

// Sum over the lanes with the same l % MR, in all of them.
template <int MR>
PGN_DEVICE float sum_beside(float x) {
  if constexpr (MR == 1) return group_sum<64>(x);
  if constexpr (MR == 4) {
    x += dpp_move<0x124>(x);  // row_ror:4
    x += dpp_move<0x128>(x);  // row_ror:8
  }
  x = swap_add<16>(x, x);
  return swap_add<32>(x, x);
}

constexpr int kWaves = 4;

// A workgroup's share: 16 RT rows (MR of each 16 read: MR = 1 or 4 where there are no more), WN NT column tiles of the
// 16 columns, WK waves sharing the contracted columns of each (WN WK = 4). Rows go to LDS in P bf16 parts, a chunk of CB
// blocks of 128 columns at a time, as the matrix core takes them; codes straight to registers, one chunk ahead.
template <class T, int P, int GS, int MR, int RT, int U, int WK, int NT>
__global__ __launch_bounds__(64 * kWaves) void linear(const T* __restrict__ x, const u32x4* __restrict__ codes,
                                                      const __bf16* __restrict__ scales, const T* __restrict__ lnw,
                                                      const T* __restrict__ lnb, float eps, const T* __restrict__ bias,
                                                      int act, const T* resid, T* y, int n, int N, int K, int KB,
                                                      int ctiles, int rblocks) {
  constexpr int WN = kWaves / WK, KL = 64 / MR, CB = U * 16 / (MR * RT), CBW = CB / WK, RW = MR * RT, CK8 = CB * 16;
  constexpr int WR = kWaves / RT;  // waves that stage the same rows
  static_assert(CBW * WK * MR * RT == U * 16 && (RT == 1 || MR == 16), "");
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[2][kWaves][MR];
  bf16x8* const buf = reinterpret_cast<bf16x8*>(smem);  // [2 chunks][P][CK8][RW]
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = l & 15, h = l >> 4, wk = w % WK, wn = w / WK;
  // workgroups of the same columns run on one XCD (their numbers differ by multiples of 8)
  int cg = blockIdx.x, rb = 0;
  if (rblocks > 1) {
    const int rest = blockIdx.x >> 3;
    rb = rest % rblocks;
    cg = rest / rblocks * 8 + (blockIdx.x & 7);
  }
  const int ct0 = cg * WN * NT + wn * NT;
  if (cg * WN * NT >= ctiles) return;
  const int nch = (KB + CB - 1) / CB;

  // staging: this thread's row, and its first 8-column piece of a chunk
  const int srt = w % RT, sm = l % MR, sk = (w / RT) * KL + l / MR;
  const T* const xr = x + (size_t)min(rb * 16 * RT + 16 * srt + sm, n - 1) * K;
  Raw<T> raw[U];
  auto load_x = [&](int c) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = 8 * (c * CK8 + sk + u * WR * KL);
      if (k < K) raw[u].load(xr + k);
      else raw[u].zero();
    }
  };
  u32x4 cw[CBW][NT];
  unsigned sw[CBW][NT][GS == 1 ? 2 : 1];
  auto load_w = [&](int j, int c) {
    const int kb = c * CB + wk + WK * j;
    if (kb >= KB) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const size_t tile = (size_t)min(ct0 + t, ctiles - 1) * KB + kb;
      cw[j][t] = codes[tile * 64 + l];
      const __bf16* sp = scales + (tile * 16 + i) * (4 / GS);
      if constexpr (GS == 1) {
        const i32x2 v = *reinterpret_cast<const i32x2*>(sp);
        sw[j][t][0] = (unsigned)v[0];
        sw[j][t][1] = (unsigned)v[1];
      } else if constexpr (GS == 2) {
        sw[j][t][0] = *reinterpret_cast<const unsigned*>(sp);
      } else {
        sw[j][t][0] = *reinterpret_cast<const unsigned short*>(sp);
      }
    }
  };
  load_x(0);
#pragma unroll
  for (int j = 0; j < CBW; ++j) load_w(j, 0);

  // the row's mean and 1 / sigma: the sum, then the squares about the mean, each over the whole row
  float mean = 0.f, rstd = 1.f;
  const bool norm = P == 2 || (P == 3 && lnw != nullptr);
  if (norm) {
    auto total = [&](auto&& f, int slot) {
      float s = 0.f;
      for (int c = 0; c < nch; ++c) {
        if (nch > 1) load_x(c);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (8 * (c * CK8 + sk + u * WR * KL) < K) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s += f(raw[u].get(e));
          }
        }
      }
      s = sum_beside<MR>(s);
      if (l < MR) red[slot][w][l] = s;
      __syncthreads();
      s = 0.f;
#pragma unroll
      for (int v = 0; v < WR; ++v) s += red[slot][srt + RT * v][sm];
      return s;
    };
    mean = total([](float v) { return v; }, 0) / (float)K;
    const float var = total([mean](float v) { return (v - mean) * (v - mean); }, 1) / (float)K;
    rstd = 1.f / sqrtf(var + eps);
    if (nch > 1) load_x(0);
  }
  auto store_x = [&](int c) {
    bf16x8* const to = buf + (size_t)(c & 1) * P * CK8 * RW;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k8 = sk + u * WR * KL, k = 8 * (c * CK8 + k8);
      bf16x8 part[P];
      if constexpr (P == 1) {
        part[0] = __builtin_bit_cast(bf16x8, raw[u].a);
      } else {
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = raw[u].get(e);
        if (norm && k < K) {
          Raw<T> g, b;
          g.load(lnw + k);
          if (lnb) b.load(lnb + k);
          else b.zero();
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = (z[e] - mean) * rstd * g.get(e) + b.get(e);
        }
        split8<P>(z, part);
      }
#pragma unroll
      for (int p = 0; p < P; ++p) to[((size_t)p * CK8 + k8) * RW + 16 * srt + sm] = part[p];
    }
  };
  store_x(0);

  f32x4 acc[RT][NT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < nch; ++c) {
    __syncthreads();
    if (c + 1 < nch) load_x(c + 1);
    const bf16x8* const from = buf + (size_t)(c & 1) * P * CK8 * RW;
#pragma unroll
    for (int j = 0; j < CBW; ++j) {
      if (c * CB + wk + WK * j < KB) {
        const bf16x8* const at = from + (size_t)((wk + WK * j) * 16 + h) * RW + i % MR;
#pragma unroll
        for (int q = 0; q < 4 / GS; ++q) {
          f32x4 d[RT][NT];
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t) d[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = q * GS; ks < (q + 1) * GS; ++ks) {
            bf16x8 b[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) b[t] = operand(cw[j][t][ks]);
#pragma unroll
            for (int p = P - 1; p >= 0; --p)  // the smallest parts first
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                const bf16x8 a = at[((size_t)p * CK8 + 4 * ks) * RW + 16 * r];
#pragma unroll
                for (int t = 0; t < NT; ++t) d[r][t] = pgn_mfma(a, b[t], d[r][t]);
              }
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const unsigned sv = sw[j][t][GS == 1 ? q >> 1 : 0];
            const float s = q & 1 ? float_of(sv & 0xffff0000u) : bf16_bits(sv);
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[r][t] += s * d[r][t];
          }
        }
      }
      if (c + 1 < nch) load_w(j, c + 1);
    }
    if (c + 1 < nch) store_x(c + 1);
  }

  auto finish = [&](float v, int row, int col) {
    if (row < n && col < N) {
      if (bias) v += (float)bias[col];
      if (act == 1) v = pgn_gelu_erf(v);
      const size_t off = (size_t)row * N + col;
      if (resid) v += (float)resid[off];
      y[off] = (T)v;
    }
  };
  const int row0 = rb * 16 * RT;
  if constexpr (WK == 1) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) finish(acc[r][t][e], row0 + 16 * r + 4 * h + e, (ct0 + t) * 16 + i);
  } else {
    // the waves' sums joined in order: wave wk's at [wk][wn][t][r][lane][e]
    __syncthreads();
    f32x4* const part = reinterpret_cast<f32x4*>(smem);
    constexpr int S = WN * NT * RT * 64;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t) part[wk * S + ((wn * NT + t) * RT + r) * 64 + l] = acc[r][t];
    __syncthreads();
    for (int o = tid; o < S * 4; o += 64 * kWaves) {
      const int e = o & 3, lane = o >> 2 & 63, r = (o >> 8) % RT, tile = (o >> 8) / RT;
      const int row = row0 + 16 * r + 4 * (lane >> 4) + e, col = (cg * WN * NT + tile) * 16 + (lane & 15);
      if (row < n && col < N) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < WK; ++k) v += reinterpret_cast<const float*>(part)[k * S * 4 + o];
        finish(v, row, col);
      }
    }
  }
}

struct Call {
  const void *x, *codes, *scales, *lnw, *lnb, *bias, *resid;
  void* y;
  float eps;
  int act, n, N, K;
  hipStream_t st;
};

template <class T, int P, int GS, int MR, int RT, int U, int WK, int NT>
int launch(const Call& a) {
  constexpr int CB = U * 16 / (MR * RT), WN = kWaves / WK;
  const int KB = (a.K + kTileCols - 1) / kTileCols, ctiles = (a.N + 15) / 16;
  const int rblocks = (a.n + 16 * RT - 1) / (16 * RT), groups = (ctiles + WN * NT - 1) / (WN * NT);
  const int64_t blocks = rblocks > 1 ? (int64_t)(groups + 7) / 8 * 8 * rblocks : groups;
  const size_t chunk = (size_t)P * U * 4096;
  const size_t lds = std::max<size_t>(KB > CB ? 2 * chunk : chunk, WK > 1 ? (size_t)kWaves * NT * RT * 1024 : 0);
  const auto fn = linear<T, P, GS, MR, RT, U, WK, NT>;
  const hipError_t e = pgn_lds_limit(reinterpret_cast<const void*>(fn), 2 * chunk);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(64 * kWaves), lds, a.st, (const T*)a.x, (const u32x4*)a.codes,
                     (const __bf16*)a.scales, (const T*)a.lnw, (const T*)a.lnb, a.eps, (const T*)a.bias, a.act,
                     (const T*)a.resid, (T*)a.y, a.n, a.N, a.K, KB, ctiles, rblocks);
  PGN_RETURN_LAUNCH();
}

template <class T, int P, int GS>
int by_rows(const Call& a) {
  if (a.n == 1) return launch<T, P, GS, 1, 1, 2, 4, 1>(a);
  if (a.n <= 4) return launch<T, P, GS, 4, 1, 4, 4, 1>(a);
  if (a.n <= 64) return launch<T, P, GS, 16, 1, 4, 2, 1>(a);
  return launch<T, P, GS, 16, 4, P == 1 ? 8 : 4, 1, P == 1 ? 4 : 2>(a);
}

template <class T, int P>
int by_group(const Call& a, int64_t group) {
  return group == 32 ? by_rows<T, P, 1>(a) : group == 64 ? by_rows<T, P, 2>(a) : by_rows<T, P, 4>(a);
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

#define PGN_BY_TYPE(FN, SRC, ...)                                                                             \
  const dim3 grid((unsigned)((tiles + 3) / 4));                                                               \
  const hipStream_t st = (hipStream_t)stream;                                                                 \
  if (bf16) {                                                                                                 \
    if (group == 32) hipLaunchKernelGGL((FN<__bf16, 1>), grid, dim3(256), 0, st, __VA_ARGS__(__bf16));        \
    else if (group == 64) hipLaunchKernelGGL((FN<__bf16, 2>), grid, dim3(256), 0, st, __VA_ARGS__(__bf16));   \
    else hipLaunchKernelGGL((FN<__bf16, 4>), grid, dim3(256), 0, st, __VA_ARGS__(__bf16));                    \
  } else {                                                                                                    \
    if (group == 32) hipLaunchKernelGGL((FN<float, 1>), grid, dim3(256), 0, st, __VA_ARGS__(float));          \
    else if (group == 64) hipLaunchKernelGGL((FN<float, 2>), grid, dim3(256), 0, st, __VA_ARGS__(float));     \
    else hipLaunchKernelGGL((FN<float, 4>), grid, dim3(256), 0, st, __VA_ARGS__(float));                      \
  }

extern "C" int pragnosia_fp4_quantize(const void* W, int bf16, void* codes, void* scales, int64_t N, int64_t K,
                                      int64_t group, void* stream) {
  PGN_CHECK_ARG(W && codes && scales && weight_ok(N, K, group) && aligned(W, codes, scales));
  const int64_t tiles = tiles_of(N, K);
  const int KB = (int)((K + kTileCols - 1) / kTileCols);
#define PGN_ARGS(T) (const T*)W, (u32x4*)codes, (__bf16*)scales, N, (int)K, KB, tiles
  PGN_BY_TYPE(quantize, W, PGN_ARGS)
#undef PGN_ARGS
  PGN_RETURN_LAUNCH();
}

extern "C" int pragnosia_fp4_dequantize(const void* codes, const void* scales, void* W, int bf16, int64_t N, int64_t K,
                                        int64_t group, void* stream) {
  PGN_CHECK_ARG(W && codes && scales && weight_ok(N, K, group) && aligned(W, codes, scales));
  const int64_t tiles = tiles_of(N, K);
  const int KB = (int)((K + kTileCols - 1) / kTileCols);
#define PGN_ARGS(T) (const u32x4*)codes, (const __bf16*)scales, (T*)W, N, (int)K, KB, tiles
  PGN_BY_TYPE(dequantize, W, PGN_ARGS)
#undef PGN_ARGS
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
  PGN_CHECK_ARG(((ya | (uintptr_t)bias | (uintptr_t)resid) & (size - 1)) == 0);
  PGN_CHECK_ARG(xa + (uintptr_t)(n * K) * size <= ya || ya + (uintptr_t)(n * N) * size <= xa);
  const Call a{x, codes, scales, ln_weight, ln_bias, bias, resid, y, ln_eps, act, (int)n, (int)N, (int)K,
               (hipStream_t)stream};
  if (!bf16) return by_group<float, 3>(a, group);
  return ln_weight ? by_group<__bf16, 2>(a, group) : by_group<__bf16, 1>(a, group);
}
