// A workgroup's bf16 matrix product over a tile of outputs, shared by the head's kernels: acc(x, y) = sum_k X(x, k)
// Y(y, k) on v_mfma_f32_16x16x32_bf16, WX x WY waves of 16 NA x 16 NB outputs each.
//
// Either operand comes in one of two layouts: with the contracted index k running along its rows in memory (KR = false:
// h, W or dl read along their rows), or down its rows (KR = true: the same matrices contracted over tokens or words).
//
// A step contracts 64 values of k, staged into one of NS LDS buffers straight from memory (buffer loads to LDS, 16
// bytes a lane). Step s, in a wave (its first half's fragments are in registers already):
//     read the second half's fragments;  multiply the first half
//     wait until stage s + 1 has arrived; barrier (every wave has read all of stage s)
//     issue the loads of stage s + NS into the buffer of stage s;  read stage s + 1's first half;  multiply the second
// so that fragment reads run beside products, one barrier a step, and a stage has NS - 1 steps to arrive. Reads and
// loads are spread among the products by hand (reads first: 5% slower; in fewer groups: 0 - 4%). Measured with 256 x
// 256 tiles at 8192^3: 1.33 - 1.36 PFLOP/s in every pair of layouts a tile a workgroup, 1.44 - 1.55 with a run of
// tiles (gemm_tiles), the library's product 1.35 and 1.18. Stages past the last are issued too, from offsets past the
// resource (zeros, no memory traffic), so that the wait counts are constants.
//
// A buffer load to LDS writes its 64 lanes' 16 bytes consecutively, so the arrangement against bank conflicts is made
// by which 16 bytes each lane fetches:
//   KR = false: an LDS row is one row's 64 k (128 bytes, eight segments of 16); segment s of row r holds k segment
//     s ^ (r % 8).
//   KR = true: an LDS row is one k's columns, in granules of 16 columns (32 bytes); granule s of row k holds granule
//     s ^ f(k), read with ds_read_b64_tr_b16. Half a read touches the rows k = 0 .. 3 and 8 .. 11 (of 16), which f
//     spreads over all banks: f = k % 4 + 4 (k / 8 % 2) where a row is a multiple of 256 bytes, and k / 2 % 2 +
//     2 (k / 8 % 2) where it is an odd multiple of 128 (odd rows then start in the other half of the banks).
// Both measured 240 - 250 bytes a clock and compute unit, the rate of consecutive reads. Within a 32-wide k block lane
// group g holds k = 8 g .. 8 g + 7 of both operands.
//
// Range checks: a buffer resource covers exactly the rows that exist, so rows past the operand read as zero; a k
// segment past the end of a row, or a column past it, is fetched from an offset past the resource (zero), whatever
// follows there.
#pragma once
#include "mfma_tile.h"

namespace pgn {

constexpr int kGemmK = 64;    // k a step
constexpr int kXcdCount = 8;  // XCDs of an MI355X, taking workgroups in turn

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) const bf16x8 lds_bf16x8;

// A matrix operand: `rows` rows of pitch `ld` elements (a multiple of 8) at p (16-byte aligned).
struct Operand {
  const __bf16* p;
  int64_t ld, rows;
};

// 16 bytes a lane from base + off (zero past `records` bytes) to LDS address lds + 16 lane; base, records and lds
// uniform. As an instruction of its own, not the builtin: before a transposing LDS read the compiler waits for every
// load to LDS that it knows of, which would leave a stage no time to arrive. No register is written, so nothing of the
// compiler's is in flight; the arrival is waited for by wait_loads, and a wait for another access only becomes
// stricter by these. (The s_nop covers the five wait states from a lane read into a scalar register to its use as a
// resource.)
PGN_DEVICE void load_to_lds(const char* base, int records, int off, unsigned lds) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const i32x4 r = {(int)(uint32_t)a, (int)((uint32_t)(a >> 32) & 0xffffu), records, 0x00020000};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(r)
               : "memory", "m0");
}

PGN_DEVICE unsigned lds_address(const void* p) { return (unsigned)(uintptr_t)(lds_void*)p; }

// One operand's staging: R rows (KR = false) or columns (KR = true) of the tile, T threads.
template <bool KR, int R, int T>
struct Stager {
  static constexpr int kBytes = R * kGemmK * 2;
  static constexpr int kLoads = kBytes / (T * 16);
  static constexpr int kRowBytes = KR ? 2 * R : 128;
  // Rows that a load of all threads covers: where they are whole and the arrangement repeats after them, a lane's
  // offset is the same for every load, from a base that moves by kLoadRows rows.
  static constexpr int kLoadRows = T * 16 / kRowBytes;
  static constexpr bool kSame = T * 16 % kRowBytes == 0 && kLoadRows % 16 == 0;
  static constexpr int kOffs = kSame ? 1 : kLoads;
  static_assert(kBytes % (T * 16) == 0, "whole loads");
  static_assert(!KR || R % 64 == 0, "the granules of a row are exchanged within aligned groups of four or eight");

  const __bf16* base;  // the tile's first row (KR = false), or row k_begin
  int64_t bytes;       // from there to the operand's end
  int64_t step;        // bytes from one stage to the next
  int pitch;           // bytes of a row
  int off[kOffs];      // a lane's bytes from base, or past any resource
  int k_seg;           // KR = false: the lane's first k in a stage

  static PGN_DEVICE int swizzle(int k) {
    return kRowBytes % 256 == 0 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2);
  }

  // The tile at x0, k from k_begin to k_end. KR = false: lanes() once, then any number of tiles.
  PGN_DEVICE void lanes(const Operand& o, int tid) {
    static_assert(!KR, "");
    k_seg = 8 * ((tid & 7) ^ ((tid >> 3) & 7));
#pragma unroll
    for (int u = 0; u < kOffs; ++u) off[u] = ((T / 8) * u + (tid >> 3)) * (int)o.ld * 2 + 2 * k_seg;
    step = kGemmK * 2;
    pitch = (int)o.ld * 2;
  }
  PGN_DEVICE void tile(const Operand& o, int64_t x0, int64_t k_begin) {
    base = o.p + x0 * o.ld + k_begin;
    bytes = (min((int64_t)R, o.rows - x0) * o.ld - k_begin) * 2;
  }
  PGN_DEVICE void init(const Operand& o, int64_t x0, int64_t k_begin, int64_t k_end, int tid) {
    if constexpr (!KR) {
      lanes(o, tid);
      tile(o, x0, k_begin);
    } else {
      base = o.p + k_begin * o.ld;
      bytes = (k_end - k_begin) * o.ld * 2;
      step = kGemmK * o.ld * 2;
      k_seg = 0;
      pitch = (int)o.ld * 2;
#pragma unroll
      for (int u = 0; u < kOffs; ++u) {
        const int e = u * T + tid, k = e / (kRowBytes / 16), s = e - k * (kRowBytes / 16);
        const int col = (int)x0 + 8 * (s ^ (2 * swizzle(k)));
        off[u] = col < (int)o.ld ? (k * (int)o.ld + col) * 2 : 0x7ffffff0;
      }
    }
  }

  // Stage s of the range [k_begin, k_end): aim() at it, then its kLoads loads into lds (wave w's share). A stage past
  // the last loads nothing.
  const char* at;
  int records, beyond;
  PGN_DEVICE void aim(int s, int64_t k_count) {
    at = reinterpret_cast<const char*>(base) + s * step;
    records = (int)max((int64_t)0, min(bytes - s * step, (int64_t)0x7fff0000));
    beyond = 0;
    if constexpr (!KR) {
      // all ones past the range's end: the offset is then past the resource
      const int room = (int)min(k_count - (int64_t)s * kGemmK, (int64_t)kGemmK);
      beyond = ((room - 1 - k_seg) >> 31) & 0x7ffffff0;
    }
  }
  template <int U>
  PGN_DEVICE void load(unsigned lds, int w) const {
    const int ahead = kSame ? U * kLoadRows * pitch : 0;
    load_to_lds(at + ahead, max(0, records - ahead), off[kSame ? 0 : U] | beyond, lds + U * T * 16 + w * 1024);
  }
};

// A wave's fragments of a staged operand: 16 rows (or columns) x0 .. of k block kb.
template <bool KR, int R>
struct Reader {
  static constexpr int kRowBytes = KR ? 2 * R : 128;
  // byte offsets; KR = false: in k block 0 (the other is 64 bytes away, by an exchange); KR = true: by granule within
  // an aligned eight (or four)
  int at[KR ? 8 : 1];

  PGN_DEVICE void init(int x0, int g, int i) {
    if constexpr (!KR) {
      at[0] = (x0 + i) * 128 + (g ^ (i & 7)) * 16;
    } else {
      const int f = kRowBytes % 256 == 0 ? (i >> 2) | ((g & 1) << 2) : ((i >> 3) & 1) | ((g & 1) << 1);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        at[q] = (8 * g + (i >> 2)) * kRowBytes + (((x0 >> 4) + q) ^ f) * 32 + 8 * (i & 3);
    }
  }

  // fragment Q: rows (columns) x0 + 16 Q ..; Q < 8. lds: address of the buffer.
  template <int Q, int KB>
  PGN_DEVICE bf16x8 get(unsigned lds) const {
    if constexpr (!KR) {
      return *(lds_bf16x8*)(lds + (KB ? at[0] ^ 64 : at[0]) + Q * 16 * 128);
    } else {
      const unsigned p = lds + at[Q] + 32 * KB * kRowBytes;
      return cat8(__builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)p),
                  __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(p + 4 * kRowBytes)));
    }
  }
};

template <int NA_, int NB_, int WX_, int WY_, int NS_>
struct Tile {
  static constexpr int NA = NA_, NB = NB_, WX = WX_, WY = WY_, NS = NS_;
  static constexpr int X = 16 * NA * WX, Y = 16 * NB * WY, kThreads = 64 * WX * WY;
  static constexpr int kStage = (X + Y) * kGemmK * 2, kLds = NS * kStage;
  static constexpr int kLdsInfo = kLds + 2 * kThreads * 16;  // with gemm_tiles' row data
  static constexpr int kLoads = kStage / (kThreads * 16);  // a thread's loads of a stage
  static_assert(kLdsInfo <= 160 * 1024 && NS >= 2, "");
};

template <int N>
PGN_DEVICE void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// Fragments of both halves of a stage, and their products.
template <class C, bool XKR, bool YKR>
struct Frags {
  static constexpr int kX = C::X * kGemmK * 2;  // bytes of X's part of a buffer
  Reader<XKR, C::X> rx;
  Reader<YKR, C::Y> ry;
  bf16x8 fx[2][C::NA], fy[2][C::NB];

  PGN_DEVICE void init(const WaveIdx& t) {
    rx.init(16 * C::NA * (t.w % C::WX), t.g, t.i), ry.init(16 * C::NB * (t.w / C::WX), t.g, t.i);
  }
  // Fragment Q of half KB: Y's, then X's.
  template <int KB, int Q>
  PGN_DEVICE void read_one(unsigned p) {
    if constexpr (Q < C::NB)
      fy[KB][Q] = ry.template get<Q, KB>(p + kX);
    else
      fx[KB][Q - C::NB] = rx.template get<Q - C::NB, KB>(p);
  }
  template <int KB>
  PGN_DEVICE void read(unsigned p) {
    static_for<0, C::NA + C::NB>([&](auto q) { read_one<KB, q.value>(p); });
  }
  // The products of half KB, NB at a time, and among them the fragments of the other half read from p and loads(u), u <
  // kLoads: the fragments before the last group, so that they have arrived when the half ends.
  template <int KB, int kLoads, class L>
  PGN_DEVICE void multiply(f32x4 (&acc)[C::NA][C::NB], unsigned p, L&& loads) {
    constexpr int kFrags = C::NA + C::NB, kGroups = C::NA > 1 ? C::NA - 1 : 1;
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this half's fragments, read during the half before
    static_for<0, C::NA>([&](auto a) {
      constexpr int A = decltype(a)::value;
      static_for<A * kLoads / C::NA, (A + 1) * kLoads / C::NA>([&](auto u) { loads(u); });
      constexpr int lo = A * kFrags / kGroups, hi = (A + 1) * kFrags / kGroups;
      static_for<(lo < kFrags ? lo : kFrags), (hi < kFrags ? hi : kFrags)>(
          [&](auto q) { read_one<1 - KB, decltype(q)::value>(p); });
#pragma unroll
      for (int b = 0; b < C::NB; ++b) acc[A][b] = pgn_mfma(fx[KB][A], fy[KB][b], acc[A][b]);
      __builtin_amdgcn_sched_barrier(0);
    });
  }
};

template <class C>
PGN_DEVICE void zero_acc(f32x4 (&acc)[C::NA][C::NB]) {
#pragma unroll
  for (int a = 0; a < C::NA; ++a)
#pragma unroll
    for (int b = 0; b < C::NB; ++b) acc[a][b] = zero4();
}

// acc[a][b]: outputs x = x0 + 16 NA wx + 16 a + 4 g + r, y = y0 + 16 NB wy + 16 b + i of wave (wx, wy) = (w % WX, w /
// WX), summed over k in [k_begin, k_end); for KR = false k_end <= ld.
template <class C, bool XKR, bool YKR>
PGN_DEVICE void gemm_tile(const Operand& X, const Operand& Y, int64_t x0, int64_t y0, int64_t k_begin, int64_t k_end,
                          unsigned char* lds, f32x4 (&acc)[C::NA][C::NB]) {
  const WaveIdx t = wave_idx();
  const int tid = threadIdx.x;
  typedef Frags<C, XKR, YKR> F;
  Stager<XKR, C::X, C::kThreads> sx;
  Stager<YKR, C::Y, C::kThreads> sy;
  sx.init(X, x0, k_begin, k_end, tid), sy.init(Y, y0, k_begin, k_end, tid);
  F f;
  f.init(t);
  const int64_t k_count = k_end - k_begin;
  const int steps = (int)((k_count + kGemmK - 1) / kGemmK);
  zero_acc<C>(acc);
  const unsigned lds0 = lds_address(lds);
  constexpr int kLx = Stager<XKR, C::X, C::kThreads>::kLoads;
  auto aim = [&](int s) { sx.aim(s, k_count), sy.aim(s, k_count); };
  auto load = [&](auto u_c, int buf) {
    constexpr int u = decltype(u_c)::value;
    const unsigned p = lds0 + buf * C::kStage;
    if constexpr (u < kLx)
      sx.template load<u>(p, t.w);
    else
      sy.template load<u - kLx>(p + F::kX, t.w);
  };
  for (int s = 0; s < C::NS; ++s) {
    aim(s);
    static_for<0, C::kLoads>([&](auto u) { load(u, s); });
  }
  wait_loads<C::kLoads * (C::NS - 1)>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  f.template read<0>(lds0);
  int buf = 0;
  for (int s = 0; s < steps; ++s) {
    const int next = buf + 1 == C::NS ? 0 : buf + 1;
    f.template multiply<0, 0>(acc, lds0 + buf * C::kStage, [](auto) {});
    aim(s + C::NS);
    wait_loads<C::kLoads * (C::NS - 2)>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    f.template multiply<1, C::kLoads>(acc, lds0 + next * C::kStage, [&](auto u) { load(u, buf); });
    buf = next;
  }
  // nothing in flight into the buffers, nothing being read: they may be used again
  wait_loads<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Workgroup `wg` runs on XCD wg % 8. An XCD takes a contiguous run of the items, its workgroups neighbours in it at any
// time, so they share operands in its L2: the items are first, first + stride, .. below end.
struct XcdRun {
  int first, stride, end;
};
PGN_DEVICE XcdRun xcd_run(int items) {
  const int per = (items + kXcdCount - 1) / kXcdCount, x = blockIdx.x % kXcdCount;
  return {x * per + (int)blockIdx.x / kXcdCount, (int)gridDim.x / kXcdCount, min(items, (x + 1) * per)};
}

// The same for a run of tiles with both operands along their rows, k from 0 to d: the run's items (at least one),
// at(item, ix, iy) giving their tiles, epilogue(acc, x0, y0, info) after each. The stages of the next tile are under
// way while a tile's last steps and its epilogue run.
//
// info: kInfo bytes of data of each of the tile's Y rows (row y's at rows + y kInfo, row_count of them; the rest reads
// as zero), copied to LDS a tile ahead: into one of two places by the tile's parity, from a tile's first barrier on,
// when the tile before, that place's last reader, is done; complete at the tile's own first barrier.
//
// kStores: how many stores every wave's epilogue issues at the least, whatever its tile holds. They need not have left
// before the next tile's first stages are read: those loads were issued before them, and memory operations are counted
// in order.
template <class C, int kInfo, int kStores, class At, class Epilogue>
PGN_DEVICE void gemm_tiles(const Operand& X, const Operand& Y, int64_t d, const void* rows, int64_t row_count,
                           const XcdRun& run, unsigned char* lds, At&& at, Epilogue&& epilogue) {
  static_assert(C::Y * kInfo <= C::kThreads * 16 && kInfo % 8 == 0, "one load a thread");
  const WaveIdx t = wave_idx();
  const int tid = threadIdx.x, steps = (int)((d + kGemmK - 1) / kGemmK);
  typedef Frags<C, false, false> F;
  Stager<false, C::X, C::kThreads> sx;
  Stager<false, C::Y, C::kThreads> sy;
  sx.lanes(X, tid), sy.lanes(Y, tid);
  F f;
  f.init(t);
  // the next stage to load: step ls of tile item `li`
  int li = run.first, ls = 0;
  auto aim = [&]() {
    int ix = 0, iy = 0;
    if (li < run.end) at(li, ix, iy);
    sx.tile(X, (int64_t)ix * C::X, 0), sy.tile(Y, (int64_t)iy * C::Y, 0);
    if (li >= run.end) sx.bytes = sy.bytes = 0;  // loads nothing
  };
  const unsigned lds0 = lds_address(lds);
  constexpr int kLx = Stager<false, C::X, C::kThreads>::kLoads;
  auto load = [&](auto u_c, int buf) {
    constexpr int u = decltype(u_c)::value;
    const unsigned p = lds0 + buf * C::kStage;
    if constexpr (u == 0) sx.aim(ls, d), sy.aim(ls, d);
    if constexpr (u < kLx)
      sx.template load<u>(p, t.w);
    else
      sy.template load<u - kLx>(p + F::kX, t.w);
    if constexpr (u == C::kLoads - 1) {
      if (++ls == steps) {
        ls = 0, li += run.stride;
        aim();
      }
    }
  };
  unsigned char* const info = lds + C::kLds;
  auto load_info = [&](int item, int place) {
    int ix = 0, iy = 0;
    if (item < run.end) at(item, ix, iy);
    const int64_t y0 = (int64_t)iy * C::Y;
    const int64_t left = item < run.end && rows != nullptr ? min((int64_t)C::Y, row_count - y0) : 0;
    load_to_lds(static_cast<const char*>(rows) + (left > 0 ? y0 * kInfo : 0), (int)(left * kInfo), tid * 16,
                lds0 + C::kLds + place * C::kThreads * 16 + t.w * 1024);
  };
  aim();
  load_info(run.first, 0);
  for (int s = 0; s < C::NS; ++s) static_for<0, C::kLoads>([&](auto u) { load(u, s); });
  wait_loads<C::kLoads * (C::NS - 1)>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  int buf = 0, place = 0;
  for (int item = run.first; item < run.end; item += run.stride) {
    int ix, iy;
    at(item, ix, iy);
    f32x4 acc[C::NA][C::NB];
    zero_acc<C>(acc);
    // The first half of step s. Stage s + 1 has arrived at its end, and every wave's reads of stage s are done. The
    // stages that were issued before the last epilogue's stores need not wait for those.
    auto half = [&](int s) {
      f.template multiply<0, 0>(acc, lds0 + buf * C::kStage, [](auto) {});
      if (steps < C::NS)  // the row data of this tile may be among the last loads
        wait_loads<0>();
      else if (s < C::NS - 1 && item != run.first)
        wait_loads<C::kLoads * (C::NS - 2) + kStores>();
      else
        wait_loads<C::kLoads * (C::NS - 2)>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (s == 0) load_info(item + run.stride, place ^ 1);
    };
    f.template read<0>(lds0 + buf * C::kStage);
    // (the last step reads the next tile's first fragments for nothing: held over the epilogue they would cost it the
    // registers, and a copy of the step without the reads costs more of them)
    for (int s = 0; s < steps; ++s) {
      half(s);
      const int next = buf + 1 == C::NS ? 0 : buf + 1;
      f.template multiply<1, C::kLoads>(acc, lds0 + next * C::kStage, [&](auto u) { load(u, buf); });
      buf = next;
    }
    epilogue(acc, (int64_t)ix * C::X, (int64_t)iy * C::Y, info + place * C::kThreads * 16);
    place ^= 1;
  }
  wait_loads<0>();
}

// Tile `item` of a grid of tx x ty tiles (x tiles, y tiles), so ordered that consecutive items share operands: bands of
// eight y tiles, within a band y fastest. In 32 bits and scalar registers (a division runs in the vector unit).
PGN_DEVICE void band_tile(int item, int tx, int ty, int& ix, int& iy) {
  constexpr unsigned kBand = 8;
  const unsigned band = (unsigned)item / (tx * kBand), y0 = band * kBand, h = min(kBand, ty - y0);
  const unsigned in = item - band * tx * kBand, x = in / h;
  ix = __builtin_amdgcn_readfirstlane(x);
  iy = __builtin_amdgcn_readfirstlane(y0 + in - x * h);
}

// Workgroups for `items` items with one each, or at most `most`, a whole number an XCD.
inline unsigned xcd_grid(int64_t items, int64_t most = (int64_t)1 << 30) {
  const int64_t per = (items + kXcdCount - 1) / kXcdCount;
  return (unsigned)((per < most / kXcdCount ? per : most / kXcdCount) * kXcdCount);
}

}  // namespace pgn
