// Rules on logits: penalties for repeated tokens, biases, masks; the processed logits, or the best token they leave
// (formulas and conventions in include/pragnosia_gen.h).
//
// One pass over the logits. A workgroup owns a tile of one row's words, whose logits it loads first. In its LDS, a 32-bit
// word each, it marks the bias entries of its words (the last of a repeated word wins, by an integer maximum) and counts
// the row's history (integer atomics: any order gives the same counts); whoever marks a word first puts it on a list. Then
// the rules go over that list, not over the words: a listed word's value is formed from its logit and left in its place.
// The pass over the tile's logits that follows takes those values, masks, and keeps the best or stores. No counts are kept
// between calls and nothing of the vocabulary's size is written but the result: a history is some kilobytes where a row of
// counts would be as large as the row of logits.
//
// Bound by the chain within a workgroup (loads, marks, settling, the pass), two of which a compute unit overlaps: one row of
// 8192 under a history of 600 4.7 us, 64 of 32768 with a history of 2000, a list of 100 and a mask 10.8, 256 bf16 rows of
// 131072 with a history of 4000, 32 entries and a mask 33.0 (4.1 TB/s of logits in and out; 21.5 without any rule).
// A row's tiles run on one XCD, whose L2 then has its history for all but the first (39.0 otherwise). Workgroups that go
// through a row's tiles by themselves, the next tile's logits on their way, took 48: their registers leave room for one.
#include <algorithm>

#include "../include/pragnosia_gen.h"
#include "argmax.h"
#include "common.h"

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u32x4;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
// A word's place in LDS: bit 31: it is in the history before `prompt`; from bit `shift` on its bias entry + 1, 0 without
// one; below its count among the rest (shift bits hold L, the rest M).
constexpr unsigned kInPrompt = 0x80000000u;
constexpr int kList = 4096;  // words of a tile that its list holds
constexpr int kAhead = 4;  // history entries a thread loads before it knows the history's length
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
  int L, M, V, words, tiles, shift;
  int rows;  // B where a row's tiles are to run on one XCD, else 0
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
PGN_DEVICE float penalised(float x, unsigned c, float r, float p, float f) {
#pragma clang fp contract(off)
  x = x > 0.f ? x / r : x * r;
  if (c) {
    x = x - p;
    const float fc = f * (float)c;
    x = x - fc;
  }
  return x;
}

// Bit e of `m` as a word of zeros or ones.
PGN_DEVICE unsigned spread(unsigned m, int e) { return (unsigned)((int)(m << (31 - e)) >> 31); }

// -infinity where `off` has a word's bit, on raw elements.
PGN_DEVICE void mask_vector(u32x4& v, unsigned off, float) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned m = spread(off, e);
    v[e] = (v[e] & ~m) | (0xff800000u & m);
  }
}
PGN_DEVICE void mask_vector(u32x4& v, unsigned off, __bf16) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned m = (spread(off, 2 * e) & 0xffffu) | (spread(off, 2 * e + 1) & 0xffff0000u);
    v[e] = (v[e] & ~m) | (0xff80ff80u & m);
  }
}

// W words to a workgroup, Q 16-byte vectors of logits a thread. Rows start at any element: the vectors lie at 16-byte
// addresses, so a row's first and last may be shared with its neighbours and are then taken element by element.
template <class T, int W, bool TOKEN>
__global__ __launch_bounds__(kThreads) void apply(const Args a) {
  constexpr int E = 16 / (int)sizeof(T), Q = W / kThreads / E;
  extern __shared__ __align__(16) unsigned smem[];  // with entries: words [W], settled [W / 32], list; with a mask its bits
  __shared__ Key key_s[kWaves];
  __shared__ int listed;
  static_assert(Q * kThreads * E == W && kWaves == 16, "the waves' keys are reduced in a row of 16 lanes");
  const int tid = threadIdx.x, V = a.V;
  int b = blockIdx.y, tile = blockIdx.x;
  if (a.rows) {  // (workgroups whose numbers differ by multiples of 8 share an XCD)
    const unsigned id = blockIdx.y * (unsigned)a.tiles + blockIdx.x, turn = id >> 3;
    b = (int)(turn / (unsigned)a.tiles * 8 + (id & 7));
    tile = (int)(turn % (unsigned)a.tiles);
    if (b >= a.rows) return;
  }
  const int64_t row = (int64_t)b * V;
  const int v0 = tile * W - (int)(row & (E - 1));  // the first vector's first word, at least -E + 1
  const T* const lr = (const T*)a.logits + row;
  T* const yr = (T*)a.out + row;
  const bool entries = a.L || a.M;

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
  const int64_t* const hr = a.history + (int64_t)b * a.history_stride;
  const int64_t* const br = a.bias_ids + (int64_t)b * a.bias_stride;
  const float* const bv = a.bias_values + (int64_t)b * a.bias_stride;
  int64_t id[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) id[u] = tid + u * kThreads < a.L ? hr[tid + u * kThreads] : -1;
  const int64_t len64 = a.lengths ? a.lengths[b] : a.L;
  const int len = (int)(len64 < 0 ? 0 : len64 > a.L ? a.L : len64);
  const int64_t pr64 = a.prompt ? a.prompt[b] : 0;
  const int prompt = (int)(pr64 < 0 ? 0 : pr64 > len ? len : pr64);
  const float r = a.repetition ? a.repetition[b] : a.r0, p = a.presence ? a.presence[b] : a.p0,
              f = a.frequency ? a.frequency[b] : a.f0;
  int64_t line = -1;
  if (a.S) line = a.state ? a.state[b] : a.S == 1 ? 0 : b;
  const bool masked = line >= 0, closed = line >= a.S && masked;

  unsigned* const word = smem;
  unsigned* const settled = smem + W;
  unsigned short* const list = reinterpret_cast<unsigned short*>(smem + W + W / 32);
  unsigned* const bits = smem + (entries ? W + W / 32 + kList / 2 : 0);
  if (entries) {
    for (int k = tid * 4; k < W + W / 32; k += kThreads * 4) *reinterpret_cast<u32x4*>(smem + k) = u32x4{0u, 0u, 0u, 0u};
    if (tid == 0) listed = 0;
  }
  const int line0 = max(v0, 0) >> 5;
  if (masked && !closed) {
    const int linen = (min(v0 + W, V) + 31) >> 5;  // (none where the tile lies past the row)
    const uint32_t* const mr = a.mask + line * a.words;
    for (int k = line0 + tid; k < linen; k += kThreads) bits[k - line0] = mr[k];
  }
  __syncthreads();
  if (entries) {
    // f(place in the tile) for an entry that lies in it
    auto within = [&](int64_t i, auto&& f) {
      const unsigned v = (unsigned)i, k = v - (unsigned)v0;
      if ((uint64_t)i >> 32 == 0 && v < (unsigned)V && k < (unsigned)W) f((int)k);
    };
    auto enlist = [&](int k, unsigned before) {
      if (before) return;  // marked already
      const int at = atomicAdd(&listed, 1);
      if (at < kList) list[at] = (unsigned short)k;
    };
    if (a.M) {
      for (int j = tid; j < a.M; j += kThreads)
        within(br[j], [&](int k) { enlist(k, atomicMax(word + k, ((unsigned)j + 1u) << a.shift)); });
      __syncthreads();
    }
    if (a.L) {
      auto count = [&](int t, int64_t i) {
        within(i, [&](int k) { enlist(k, t < prompt ? atomicOr(word + k, kInPrompt) : atomicAdd(word + k, 1u)); });
      };
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (tid + u * kThreads < len) count(tid + u * kThreads, id[u]);
      for (int t = tid + kAhead * kThreads; t < len; t += kThreads) count(t, hr[t]);
      __syncthreads();
    }
    auto settle = [&](int k) {
      const unsigned w = word[k], c = w & ((1u << a.shift) - 1u), e = (w & ~kInPrompt) >> a.shift;
      float z = (float)lr[v0 + k];
      if (c || (w & kInPrompt)) z = penalised(z, c, r, p, f);
      if (e) z += bv[e - 1];
      word[k] = __builtin_bit_cast(unsigned, z);
      atomicOr(settled + (k >> 5), 1u << (k & 31));
    };
    const int n = listed;
    if (n <= kList) {
      for (int j = tid; j < n; j += kThreads) settle(list[j]);
    } else {  // more words than the list holds: all that are marked
      for (int k = tid; k < W; k += kThreads)
        if (word[k]) settle(k);
    }
    __syncthreads();
  }

  float best = -__builtin_inff();
  int best_v = -1, nan_v = -1;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int k0 = (q * kThreads + tid) * E, v = v0 + k0;
    if (v >= V) continue;
    const int from = max(-v, 0), to = min(V - v, E);  // the vector's words in the row
    const unsigned set = entries ? settled[k0 >> 5] >> (k0 & 31) & ((1u << E) - 1u) : 0u;
    // one bit a masked word
    unsigned off = 0u;
    if (closed) {
      off = ~0u;
    } else if (masked) {
      const int u = max(v, 0), w0 = (u >> 5) - line0, w1 = ((v + to - 1) >> 5) - line0;
      off = ~((unsigned)(((uint64_t)bits[w1] << 32 | bits[w0]) >> (u & 31)) << from);
    }
    if constexpr (TOKEN) {
      off |= ~((1u << to) - (1u << from));
      float z[E], most = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] = element<T>(x[q], e);
      if (set) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (set >> e & 1u) z[e] = __builtin_bit_cast(float, word[k0 + e]);
      }
      bool nan = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const unsigned m = spread(off, e);
        z[e] = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, z[e]) & ~m) | (0xff800000u & m));
        nan |= z[e] != z[e];
        most = fmaxf(most, z[e]);
      }
      if (nan && nan_v < 0) {
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
          if (z[e] != z[e]) nan_v = v + e;
      }
      if (most > best) {  // words ascend, so the first among equals stays
        best = most;
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
          if (z[e] == most) best_v = v + e;
      }
    } else {
      if (set) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (set >> e & 1u) set_element(__builtin_bit_cast(float, word[k0 + e]), x[q], e, T());
      }
      mask_vector(x[q], off, T());
      if (from == 0 && to == E) {
        *reinterpret_cast<u32x4*>(yr + v) = x[q];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e >= from && e < to) yr[v + e] = (T)element<T>(x[q], e);
      }
    }
  }
  if constexpr (TOKEN) {
    if (nan_v >= 0) best_v = nan_v;
    const Key k = max_wave(Key{nan_v >= 0 ? 0xffffffffu : order_key(best), ~(unsigned)best_v});
    if ((tid & 63) == 0) key_s[tid >> 6] = k;
    __syncthreads();
    const Key all = max_row(key_s[tid & (kWaves - 1)]);
    if (tid == 0) {
      if (a.tiles == 1) a.tokens[b] = (int)~all.lo;
      else a.part[(int64_t)b * a.tiles + tile] = (uint64_t)all.hi << 32 | all.lo;
    }
  }
}

// The best of a row's tiles, one wave a row: a launch of its own, as a workgroup that waited for the others or found itself the
// last would need a counter that some call had cleared.
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

// A row's tiles of `words` words; it may start E - 1 words into a vector.
template <class T>
int64_t tiles_of(int64_t V, int words) {
  const int E = 16 / (int)sizeof(T);
  return (V + (V % E ? E - 1 : 0) + words - 1) / words;
}

int bit_length(int64_t v) {
  int n = 0;
  for (; v > 0; v >>= 1) ++n;
  return n;
}

template <class T, int W, bool TOKEN>
int launch(Args a, int64_t B, hipStream_t st) {
  constexpr size_t marks = (size_t)(W + W / 32 + kList / 2) * 4, masks = (size_t)(W / 32 + 4) * 4;
  const size_t lds = (a.L || a.M ? marks : 0) + (a.S ? masks : 0);
  a.tiles = (int)tiles_of<T>(a.V, W);
  const auto fn = apply<T, W, TOKEN>;
  if (lds > 60 << 10) {  // (what a launch may ask for without raising the kernel's limit, with key_s to spare)
    const hipError_t e = pgn_lds_limit(reinterpret_cast<const void*>(fn), marks + masks);
    if (e != hipSuccess) return (int)e;
  }
  // (rows that leave an XCD one more than another only where there are many: 65 rows of 131072 13.4 us, else 15.1)
  const bool by_row = a.L && a.tiles > 1 && (B % 8 == 0 || (B >= 64 && B < 65528));
  a.rows = by_row ? (int)B : 0;
  hipLaunchKernelGGL(fn, dim3((unsigned)a.tiles, (unsigned)(by_row ? (B + 7) / 8 * 8 : B)), dim3(kThreads), lds, st, a);
  if (TOKEN && a.tiles > 1) {
    const hipError_t f = hipGetLastError();
    if (f != hipSuccess) return (int)f;
    hipLaunchKernelGGL(pick, dim3((unsigned)B), dim3(64), 0, st, a.part, a.tiles, a.tokens);
  }
  PGN_RETURN_LAUNCH();
}

// The words of a tile. A row whose token comes from one tile takes no second launch, which is worth more than the smaller
// tiles' spread over the chip: 64 rows of 32768 with a history, a list and a mask 15.7 us eager in one tile a row, 18.0 in
// four, though alone on the GPU 10.8 against 8.1. Longer rows, and logits for a sampler: 16384 words where that leaves two
// workgroups a compute unit (256 rows of 131072 bf16: 33.0 us, with 8192 words 42.3, with 32768 38.7), else 8192.
template <class T, bool TOKEN>
int run(const Args& a, int64_t B, hipStream_t st) {
  if (TOKEN && tiles_of<T>(a.V, 8192) > 1) {
    if (tiles_of<T>(a.V, 16384) == 1) return launch<T, 16384, TOKEN>(a, B, st);
    if (tiles_of<T>(a.V, 32768) == 1) return launch<T, 32768, TOKEN>(a, B, st);
  }
  return tiles_of<T>(a.V, 16384) * B >= 512 ? launch<T, 16384, TOKEN>(a, B, st) : launch<T, 8192, TOKEN>(a, B, st);
}

// What follows a chosen token, one workgroup a row: the token joins the row's history and moves its grammar's state, and
// (emb) what decode_tail does after its argmax: the token written out, the position advanced, the next step's input. Choosing
// and this take a step 3 to 8 us more than decode_tail's argmax (one launch more).
constexpr int kTailThreads = 256;

struct Tail {
  const int64_t* tokens;
  int64_t* history;
  int64_t history_stride, cap;
  int64_t* lengths;
  const int32_t* next;
  int64_t S, V;
  int64_t* state;
  const float *emb, *pemb;
  int d, ctx;
  const int64_t* ctr_in;
  int64_t* ctr_out;
  const int64_t* pos_in;
  int64_t* pos_out;
  int64_t* out;
  int64_t n_rows;
  int64_t* tok;
  float* h;
  float* p0s;
  int L, B;
};

__global__ __launch_bounds__(kTailThreads) void tail(const Tail a) {
  const int b = blockIdx.x, tid = threadIdx.x;
  const int64_t t = a.tokens[b];
  const bool known = t >= 0 && t < a.V;
  if (tid == 0 && known) {
    if (a.lengths) {
      const int64_t n = a.lengths[b];
      if (n >= 0 && n < a.cap) {
        a.history[b * a.history_stride + n] = t;
        a.lengths[b] = n + 1;
      }
    }
    if (a.state) {
      const int64_t s = a.state[b];
      if (s >= 0 && s < a.S) a.state[b] = a.next[s * a.V + t];
    }
  }
  if (!a.emb) return;
  const int64_t c = *a.ctr_in, p = (*a.pos_in + 1) % a.ctx;
  if (tid == 0) {
    a.tok[b] = t;
    if (c >= 0 && c < a.n_rows) a.out[c * a.B + b] = t;
  }
  const float* const er = a.emb + (known ? t : 0) * a.d;
  const float* const pr = a.pemb + p * a.d;
  float* const hr = a.h + (int64_t)b * a.d;
  for (int k = tid; k < a.d; k += kTailThreads) hr[k] = (known ? er[k] : 0.f) + pr[k];
  if (b == 0) {
    if (tid == 0) {
      *a.pos_out = p;
      *a.ctr_out = c + 1;
    }
    for (int k = tid; k < a.L; k += kTailThreads) a.p0s[k] = 1.f;
  }
}

bool sizes_ok(int64_t B, int64_t V) {
  return B >= 0 && B <= 65535 && V > 0 && V <= ((int64_t)1 << 26) && B * V < ((int64_t)1 << 40);
}

}  // namespace

extern "C" int64_t pragnosia_rules_workspace_bytes(int64_t B, int64_t V) {
  if (!sizes_ok(B, V)) return PRAGNOSIA_ERR_INVALID_ARGUMENT;
  // (the most tiles that either type has; bf16 rows may start furthest into a vector)
  return V + 7 > 32768 ? (V + 7 + 8191) / 8192 * B * (int64_t)sizeof(uint64_t) : 0;
}

extern "C" int pragnosia_rules(const void* logits, int bf16, const int64_t* history, int64_t history_stride, int64_t L,
                               const int64_t* lengths, const int64_t* prompt, const float* repetition,
                               float repetition_value, const float* presence, float presence_value,
                               const float* frequency, float frequency_value, const int64_t* bias_ids,
                               const float* bias_values, int64_t M, int64_t bias_stride, const uint32_t* mask, int64_t S,
                               const int64_t* state, void* out, int64_t* tokens, void* workspace,
                               int64_t workspace_bytes, int64_t B, int64_t V, void* stream) {
  PGN_CHECK_ARG(sizes_ok(B, V) && L >= 0 && L <= ((int64_t)1 << 24) && M >= 0 && M <= ((int64_t)1 << 20) && S >= 0);
  PGN_CHECK_ARG(!out != !tokens && (L == 0 || (history && history_stride >= L)) && (repetition || repetition_value != 0.f));
  PGN_CHECK_ARG(M == 0 || (bias_ids && bias_values && (bias_stride == 0 || bias_stride >= M)));
  PGN_CHECK_ARG(bit_length(L) + bit_length(M) <= 31);
  PGN_CHECK_ARG(S == 0 || (mask && (state || S == 1 || S == B)));
  const int64_t need = tokens ? pragnosia_rules_workspace_bytes(B, V) : 0;
  PGN_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0));
  if (B == 0) return PRAGNOSIA_OK;
  PGN_CHECK_ARG(logits && (((uintptr_t)logits | (uintptr_t)out) & 15) == 0);
  const uintptr_t la = (uintptr_t)logits, oa = (uintptr_t)out, size = (uintptr_t)(B * V) * (bf16 ? 2 : 4);
  PGN_CHECK_ARG(!out || la == oa || la + size <= oa || oa + size <= la);
  const Args a{logits, history, history_stride, lengths, prompt, repetition, presence, frequency, repetition_value,
               presence_value, frequency_value, bias_ids, bias_values, bias_stride, mask, S, state, out, tokens,
               (uint64_t*)workspace, (int)L, (int)M, (int)V, (int)((V + 31) / 32), 0, bit_length(L), 0};
  const hipStream_t st = (hipStream_t)stream;
  if (tokens) return bf16 ? run<__bf16, true>(a, B, st) : run<float, true>(a, B, st);
  return bf16 ? run<__bf16, false>(a, B, st) : run<float, false>(a, B, st);
}

extern "C" int pragnosia_rules_tail(const int64_t* tokens, int64_t* history, int64_t history_stride, int64_t cap,
                                    int64_t* lengths, const int32_t* next, int64_t S, int64_t* state, const float* emb,
                                    const float* pemb, int64_t d, int64_t ctx, const int64_t* ctr_in, int64_t* ctr_out,
                                    const int64_t* pos_in, int64_t* pos_out, int64_t* out, int64_t n_rows, int64_t* tok,
                                    float* h, float* p0s, int64_t L, int64_t B, int64_t V, void* stream) {
  PGN_CHECK_ARG(sizes_ok(B, V) && (!history == !lengths) && (!history || (cap > 0 && history_stride >= cap)));
  PGN_CHECK_ARG((!next == !state) && (!next || (S > 0 && S * V < ((int64_t)1 << 40))));
  PGN_CHECK_ARG(history || next || emb);
  if (emb) {
    PGN_CHECK_ARG(pemb && ctr_in && ctr_out && pos_in && pos_out && out && tok && h && d > 0 && d < (1 << 30) && ctx > 0 &&
                  ctx < (1 << 30) && n_rows > 0 && L >= 0 && L < (1 << 30) && (L == 0 || p0s));
    PGN_CHECK_ARG(ctr_in != ctr_out && pos_in != pos_out && tok != tokens);
  }
  if (B == 0) return PRAGNOSIA_OK;
  PGN_CHECK_ARG(tokens);
  const Tail a{tokens, history, history_stride, cap, lengths, next, S, V, state, emb, pemb, (int)d, (int)ctx, ctr_in,
               ctr_out, pos_in, pos_out, out, n_rows, tok, h, p0s, (int)L, (int)B};
  hipLaunchKernelGGL(tail, dim3((unsigned)B), dim3(kTailThreads), 0, (hipStream_t)stream, a);
  PGN_RETURN_LAUNCH();
}
