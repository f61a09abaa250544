// Rules on logits: penalties for repeated tokens, biases, masks; the processed logits, or the best token they leave
// (formulas and conventions in include/pragnosia_gen.h).
//
// One pass over the logits. A workgroup owns a tile of one row's words; it counts the row's history in its LDS (integer
// atomics: any order gives the same counts), marks the bias entries of its words (the last of a repeated word wins, by an
// integer maximum), and applies the rules to logits it loaded before all that. No counts are kept between calls and
// nothing of the vocabulary's size is written but the result: a history is some kilobytes where a row of counts would be
// as large as the row of logits.
#include <algorithm>

#include "../include/pragnosia_gen.h"
#include "argmax.h"
#include "common.h"

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u32x4;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr unsigned kInPrompt = 0x80000000u;  // of a word's count: it is in the part before `prompt`
constexpr unsigned kNothing = 0x007fffffu;   // order_key(-inf): what a word has to exceed

struct Args {
  const void* logits;
  const int64_t* history;
  int64_t history_stride;
  const int64_t *lengths, *prompt;
  const float *repetition, *presence, *frequency;
  float r0, p0, f0;
  const int64_t* bias_ids;
  const float* bias_values;
  int64_t bias_stride;
  const uint32_t* mask;
  int64_t S;
  const int64_t* state;
  void* out;
  int64_t* tokens;
  uint64_t* part;  // the best key of each row's tiles, hi above lo
  int L, M, V, words, tiles;
};

template <class T>
PGN_DEVICE float element(const u32x4& v, int e);
template <>
PGN_DEVICE float element<float>(const u32x4& v, int e) {
  return __builtin_bit_cast(float, (unsigned)v[e]);
}
template <>
PGN_DEVICE float element<__bf16>(const u32x4& v, int e) {
  const unsigned u = v[e >> 1];
  return __builtin_bit_cast(float, e & 1 ? u & 0xffff0000u : u << 16);
}
PGN_DEVICE void set_element(float x, u32x4& v, int e, float) { v[e] = __builtin_bit_cast(unsigned, x); }
PGN_DEVICE void set_element(float x, u32x4& v, int e, __bf16) {
  const unsigned u = __builtin_bit_cast(unsigned short, pgn_bf16(x));
  v[e >> 1] = e & 1 ? (v[e >> 1] & 0xffffu) | u << 16 : (v[e >> 1] & 0xffff0000u) | u;
}

// Each operation rounded by itself.
PGN_DEVICE float penalised(float x, unsigned count, float r, float p, float f) {
#pragma clang fp contract(off)
  x = x > 0.f ? x / r : x * r;
  const unsigned c = count & ~kInPrompt;
  if (c) {
    x = x - p;
    const float fc = f * (float)c;
    x = x - fc;
  }
  return x;
}

// Q 16-byte vectors of logits a thread. Rows start at any element: the vectors lie at 16-byte addresses, so a row's first
// and last may be shared with its neighbours and are then taken element by element.
template <class T, int Q>
__global__ __launch_bounds__(kThreads) void apply(const Args a) {
  constexpr int E = 16 / (int)sizeof(T), TILE = kThreads * Q * E;
  extern __shared__ __align__(16) unsigned smem[];  // counts [TILE] with a history, bias entries [TILE] with a list, mask
  __shared__ Key key_s[kWaves];
  static_assert(kWaves == 16, "the waves' keys are reduced in a row of 16 lanes");
  const int tid = threadIdx.x, b = blockIdx.y, V = a.V;
  const int64_t row = (int64_t)b * V;
  const int v0 = (int)blockIdx.x * TILE - (int)(row & (E - 1));  // the first vector's first word, at least -E + 1
  const T* const lr = (const T*)a.logits + row;
  T* const yr = (T*)a.out + row;

  u32x4 x[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int v = v0 + (q * kThreads + tid) * E;
    x[q] = u32x4{0u, 0u, 0u, 0u};
    if (v >= 0 && v + E <= V) {
      x[q] = *reinterpret_cast<const u32x4*>(lr + v);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v + e >= 0 && v + e < V) set_element((float)lr[v + e], x[q], e, T());
    }
  }
  int64_t len64 = a.lengths ? a.lengths[b] : a.L;
  const int len = (int)(len64 < 0 ? 0 : len64 > a.L ? a.L : len64);
  int64_t pr64 = a.prompt ? a.prompt[b] : 0;
  const int prompt = (int)(pr64 < 0 ? 0 : pr64 > len ? len : pr64);
  const float r = a.repetition ? a.repetition[b] : a.r0, p = a.presence ? a.presence[b] : a.p0,
              f = a.frequency ? a.frequency[b] : a.f0;
  int64_t line = -1;
  if (a.S) line = a.state ? a.state[b] : a.S == 1 ? 0 : b;
  const bool masked = line >= 0, closed = line >= a.S && masked;

  unsigned* const count = smem;
  unsigned* const entry = smem + (a.L ? TILE : 0);
  unsigned* const bits = entry + (a.M ? TILE : 0);
  const int arrays = (a.L ? TILE : 0) + (a.M ? TILE : 0);
  for (int k = tid * 4; k < arrays; k += kThreads * 4) *reinterpret_cast<u32x4*>(smem + k) = u32x4{0u, 0u, 0u, 0u};
  const int word0 = max(v0, 0) >> 5;
  if (masked && !closed) {
    const int wordn = (min(v0 + TILE, V) + 31) >> 5;  // (none where the tile lies past the row)
    const uint32_t* const mr = a.mask + line * a.words;
    for (int k = word0 + tid; k < wordn; k += kThreads) bits[k - word0] = mr[k];
  }
  __syncthreads();
  if (a.L) {
    const int64_t* const hr = a.history + (int64_t)b * a.history_stride;
    for (int t0 = tid; t0 < len; t0 += kThreads * 4) {
      int64_t id[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) id[u] = t0 + u * kThreads < len ? hr[t0 + u * kThreads] : -1;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t k = id[u] - v0;
        if (id[u] >= 0 && id[u] < V && k >= 0 && k < TILE) {
          if (t0 + u * kThreads < prompt) atomicOr(count + k, kInPrompt);
          else atomicAdd(count + k, 1u);
        }
      }
    }
  }
  if (a.M) {
    const int64_t* const br = a.bias_ids + (int64_t)b * a.bias_stride;
    for (int j = tid; j < a.M; j += kThreads) {
      const int64_t id = br[j], k = id - v0;
      if (id >= 0 && id < V && k >= 0 && k < TILE) atomicMax(entry + k, (unsigned)j + 1u);
    }
  }
  __syncthreads();

  const float* const bv = a.bias_values + (int64_t)b * a.bias_stride;
  unsigned best = kNothing;
  int at = -1;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int k0 = (q * kThreads + tid) * E, v = v0 + k0;
    if (v >= V) continue;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float z = element<T>(x[q], e);
      if (a.L) {
        const unsigned c = count[k0 + e];
        if (c) z = penalised(z, c, r, p, f);
      }
      if (a.M) {
        const unsigned j = entry[k0 + e];
        if (j) z += bv[j - 1];
      }
      const int ve = v + e;
      if (masked && ve >= 0 && ve < V && (closed || !(bits[(ve >> 5) - word0] >> (ve & 31) & 1u))) z = -__builtin_inff();
      if (ve >= 0 && ve < V) {
        const unsigned key = order_key(z);
        if (key > best) {  // words ascend, so the first among equals stays
          best = key;
          at = ve;
        }
      }
      set_element(z, x[q], e, T());
    }
    if (a.out) {
      if (v >= 0 && v + E <= V) {
        *reinterpret_cast<u32x4*>(yr + v) = x[q];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (v + e >= 0 && v + e < V) yr[v + e] = (T)element<T>(x[q], e);
      }
    }
  }
  if (!a.tokens) return;
  const Key k = max_wave(Key{best, ~(unsigned)at});
  if ((tid & 63) == 0) key_s[tid >> 6] = k;
  __syncthreads();
  const Key all = max_row(key_s[tid & 15]);
  if (tid == 0) {
    if (a.tiles == 1) a.tokens[b] = (int)~all.lo;
    else a.part[(int64_t)b * a.tiles + blockIdx.x] = (uint64_t)all.hi << 32 | all.lo;
  }
}

// The best of a row's tiles, one wave a row.
__global__ __launch_bounds__(64) void pick(const uint64_t* __restrict__ part, int tiles, int64_t* __restrict__ tokens) {
  const uint64_t* const row = part + (int64_t)blockIdx.x * tiles;
  Key k{kNothing, 0u};
  for (int t = threadIdx.x; t < tiles; t += 64) {
    const uint64_t v = row[t];
    const unsigned lo = (unsigned)v, hi = (unsigned)(v >> 32);
    const bool take = hi > k.hi || (hi == k.hi && lo > k.lo);
    k.hi = take ? hi : k.hi;
    k.lo = take ? lo : k.lo;
  }
  k = max_wave(k);
  if (threadIdx.x == 0) tokens[blockIdx.x] = (int)~k.lo;
}

// Words of a tile with Q vectors a thread: 16384 at most (counts and entries are 128 KB of LDS then)
template <class T>
constexpr int tile_words(int Q) { return kThreads * Q * (16 / (int)sizeof(T)); }
template <class T>
constexpr int kMostQ = sizeof(T) == 4 ? 4 : 2;
constexpr int kMostWords = tile_words<float>(4);
static_assert(kMostWords == tile_words<__bf16>(kMostQ<__bf16>), "");

// A row's tiles; it may start E - 1 words into a vector.
template <class T>
int64_t tiles_of(int64_t V, int Q) {
  const int E = 16 / (int)sizeof(T);
  return (V + (V % E ? E - 1 : 0) + tile_words<T>(Q) - 1) / tile_words<T>(Q);
}

// Vectors a thread: one tile where the row fits one (no second launch), else the largest tile that leaves two workgroups a
// compute unit (each reads its row's whole history).
template <class T>
int vectors(int64_t B, int64_t V) {
  for (int Q = 1; Q <= kMostQ<T>; Q *= 2)
    if (tiles_of<T>(V, Q) == 1) return Q;
  int Q = kMostQ<T>;
  while (Q > 1 && tiles_of<T>(V, Q) * B < 512) Q /= 2;
  return Q;
}

template <class T, int Q>
int launch(const Args& a, int64_t B, hipStream_t st) {
  constexpr int tile = tile_words<T>(Q);
  const size_t lds = ((size_t)(a.L ? tile : 0) + (a.M ? tile : 0) + (a.S ? tile / 32 + 4 : 0)) * 4;
  const auto fn = apply<T, Q>;
  const hipError_t e = pgn_lds_limit(reinterpret_cast<const void*>(fn), (size_t)(2 * tile + tile / 32 + 4) * 4);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(fn, dim3((unsigned)a.tiles, (unsigned)B), dim3(kThreads), lds, st, a);
  if (a.tokens && a.tiles > 1) {
    const hipError_t f = hipGetLastError();
    if (f != hipSuccess) return (int)f;
    hipLaunchKernelGGL(pick, dim3((unsigned)B), dim3(64), 0, st, a.part, a.tiles, a.tokens);
  }
  PGN_RETURN_LAUNCH();
}

template <class T>
int run(Args a, int64_t B, hipStream_t st) {
  const int Q = vectors<T>(B, a.V);
  a.tiles = (int)tiles_of<T>(a.V, Q);
  if (Q == 1) return launch<T, 1>(a, B, st);
  if (Q == 2) return launch<T, 2>(a, B, st);
  return launch<T, kMostQ<T>>(a, B, st);
}

bool sizes_ok(int64_t B, int64_t V) {
  return B >= 0 && B <= 65535 && V > 0 && V <= ((int64_t)1 << 26) && B * V < ((int64_t)1 << 40);
}

}  // namespace

extern "C" int64_t pragnosia_rules_workspace_bytes(int64_t B, int64_t V) {
  if (!sizes_ok(B, V)) return PRAGNOSIA_ERR_INVALID_ARGUMENT;
  // (for either type: the most tiles are the smallest, fp32's, with the most that a row's start can be off, bf16's)
  return V + 7 > kMostWords ? (V + 7 + tile_words<float>(1) - 1) / tile_words<float>(1) * B * (int64_t)sizeof(uint64_t) : 0;
}

extern "C" int pragnosia_rules(const void* logits, int bf16, const int64_t* history, int64_t history_stride, int64_t L,
                               const int64_t* lengths, const int64_t* prompt, const float* repetition,
                               float repetition_value, const float* presence, float presence_value,
                               const float* frequency, float frequency_value, const int64_t* bias_ids,
                               const float* bias_values, int64_t M, int64_t bias_stride, const uint32_t* mask, int64_t S,
                               const int64_t* state, void* out, int64_t* tokens, void* workspace,
                               int64_t workspace_bytes, int64_t B, int64_t V, void* stream) {
  PGN_CHECK_ARG(sizes_ok(B, V) && L >= 0 && L <= ((int64_t)1 << 24) && M >= 0 && M <= ((int64_t)1 << 20) && S >= 0);
  PGN_CHECK_ARG((out || tokens) && (L == 0 || (history && history_stride >= L)) && (repetition || repetition_value != 0.f));
  PGN_CHECK_ARG(M == 0 || (bias_ids && bias_values && (bias_stride == 0 || bias_stride >= M)));
  PGN_CHECK_ARG(S == 0 || (mask && (state || S == 1 || S == B)));
  const int64_t need = tokens ? pragnosia_rules_workspace_bytes(B, V) : 0;
  PGN_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0));
  if (B == 0) return PRAGNOSIA_OK;
  PGN_CHECK_ARG(logits && (((uintptr_t)logits | (uintptr_t)out) & 15) == 0);
  const uintptr_t la = (uintptr_t)logits, oa = (uintptr_t)out, size = (uintptr_t)(B * V) * (bf16 ? 2 : 4);
  PGN_CHECK_ARG(!out || la == oa || la + size <= oa || oa + size <= la);
  const Args a{logits, history, history_stride, lengths, prompt, repetition, presence, frequency, repetition_value,
               presence_value, frequency_value, bias_ids, bias_values, bias_stride, mask, S, state, out, tokens,
               (uint64_t*)workspace, (int)L, (int)M, (int)V, (int)((V + 31) / 32), 0};
  return bf16 ? run<__bf16>(a, B, (hipStream_t)stream) : run<float>(a, B, (hipStream_t)stream);
}
