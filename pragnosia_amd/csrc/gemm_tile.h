// A workgroup's bf16 matrix product over a tile of outputs, shared by the head's kernels: acc(x, y) = sum_k X(x, k) Y(y, k)
// for 256 x 256 outputs, 8 waves of 128 x 64, v_mfma_f32_16x16x32_bf16.
//
// Either operand comes in one of two layouts: with the contracted index k running along its rows in memory (KR = false:
// h, W or dl read along their rows), or down its rows (KR = true: the same matrices contracted over tokens or words).
// Each step stages 64 values of k of both operands (32 KB each) into one of two LDS buffers, straight from memory
// (buffer loads to LDS, 16 bytes a lane), while the other buffer is multiplied: one barrier a step, and the loads of a
// step have the whole step before it to arrive.
//
// A buffer load to LDS writes its 64 lanes' 16 bytes consecutively, so the arrangement against bank conflicts is made by
// which 16 bytes each lane fetches:
//   KR = false: an LDS row is one row's 64 k (128 bytes, eight segments of 16); segment s of row r holds k segment
//     s ^ (r / 2 % 8), so that the 16 rows a fragment read touches spread over all segments.
//   KR = true: an LDS row is one k's 256 columns (512 bytes, 16 granules of 32); granule s of row k holds columns
//     16 (s ^ f(k)).., f(k) = k % 4 + 4 (k / 8 % 2): the eight rows that half a transposing read touches (k = 8 g +
//     0 .. 3 for two values of g) lie in eight granules. Read with ds_read_b64_tr_b16.
// Within a 32-wide k block lane group g holds k = 8 g .. 8 g + 7 of both operands.
//
// Range checks: a buffer resource covers exactly the rows that exist, so rows past the operand read as zero; a k segment
// past the end of a row is fetched from an offset past the resource (zero) for both operands, whatever follows there.
#pragma once
#include "mfma_tile.h"

namespace pgn {

constexpr int kGemmTile = 256;      // outputs a side
constexpr int kGemmK = 64;          // k a step
constexpr int kGemmStage = kGemmTile * kGemmK * 2;  // bytes of one operand's buffer
constexpr int kGemmLds = 4 * kGemmStage;
constexpr int kGemmThreads = 512;
constexpr int kXcdCount = 8;        // XCDs of an MI355X, taking workgroups in turn

typedef __attribute__((address_space(3))) void lds_ptr_t;

// A matrix operand: `rows` rows of pitch `ld` elements (a multiple of 8) at p (16-byte aligned).
struct Operand {
  const __bf16* p;
  int64_t ld, rows;
};

// The 64 x 256 or 256 x 64 block of `o` that a step contracts: KR = false: rows x0 .., k columns k0 .. (those below
// k_end); KR = true: k rows k0 .. (below k_end, itself at most o.rows), columns x0 ...
template <bool KR>
PGN_DEVICE void stage_operand(const Operand& o, int64_t x0, int64_t k0, int64_t k_end, unsigned char* lds, int tid) {
  constexpr int kBeyond = 0x7ffffff0;  // past any resource
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if constexpr (!KR) {
    const int64_t left = min((int64_t)kGemmTile, o.rows - x0);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<__bf16*>(o.p + x0 * o.ld), (short)0, (int)(left * o.ld * 2), 0x00020000);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = 64 * u + (tid >> 3), seg = (tid & 7) ^ ((tid >> 4) & 7);
      const int k = (int)k0 + 8 * seg;
      const int off = k < (int)k_end ? row * (int)o.ld * 2 + 2 * k : kBeyond;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t*)(lds + u * 8192 + w * 1024), 16, off, 0, 0, 0);
    }
  } else {
    const int64_t left = min((int64_t)kGemmK, k_end - k0);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<__bf16*>(o.p + k0 * o.ld), (short)0, (int)(left * o.ld * 2), 0x00020000);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = 16 * u + (tid >> 5), s = tid & 31;
      const int f = (k & 3) | ((k >> 1) & 4);
      const int col = (int)x0 + 8 * (s ^ (2 * f));
      const int off = col < (int)o.ld ? (k * (int)o.ld + col) * 2 : kBeyond;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t*)(lds + u * 8192 + w * 1024), 16, off, 0, 0, 0);
    }
  }
}

// Fragment of 16 rows x0 .. x0 + 15 of an operand for k block kb (32 wide) of a staged buffer.
template <bool KR>
PGN_DEVICE bf16x8 staged_frag(const unsigned char* lds, int x0, int kb, int g, int i) {
  if constexpr (!KR) {
    return *reinterpret_cast<const bf16x8*>(lds + (x0 + i) * 128 + ((4 * kb + g) ^ ((i >> 1) & 7)) * 16);
  } else {
    const int f = (i >> 2) | ((g & 1) << 2);
    const unsigned char* q = lds + (32 * kb + 8 * g + (i >> 2)) * 512 + (((x0 >> 4) ^ f) * 32) + 8 * (i & 3);
    return cat8(ds_read_tr(reinterpret_cast<const __bf16*>(q)), ds_read_tr(reinterpret_cast<const __bf16*>(q + 2048)));
  }
}

// acc[a][b] (a < 8, b < 4): outputs x = x0 + 128 wx + 16 a + 4 g + r, y = y0 + 64 wy + 16 b + i of wave (wx, wy) =
// (w % 2, w / 2), summed over k in [k_begin, k_end); k_begin a multiple of 64 (for KR = false also k_end <= ld).
template <bool XKR, bool YKR>
PGN_DEVICE void gemm_tile(const Operand& X, const Operand& Y, int64_t x0, int64_t y0, int64_t k_begin, int64_t k_end,
                          unsigned char* lds, f32x4 (&acc)[8][4]) {
  const WaveIdx t = wave_idx();
  const int wx = t.w & 1, wy = t.w >> 1, tid = threadIdx.x;
#pragma unroll
  for (int a = 0; a < 8; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = zero4();
  const int steps = (int)((k_end - k_begin + kGemmK - 1) / kGemmK);
  auto stage = [&](int s) {
    unsigned char* buf = lds + (s & 1) * kGemmStage;
    stage_operand<XKR>(X, x0, k_begin + (int64_t)s * kGemmK, k_end, buf, tid);
    stage_operand<YKR>(Y, y0, k_begin + (int64_t)s * kGemmK, k_end, buf + 2 * kGemmStage, tid);
  };
  if (steps > 0) stage(0);
  for (int s = 0; s < steps; ++s) {
    // this step's loads have arrived and every wave's reads of the other buffer are done
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 1 < steps) stage(s + 1);
    const unsigned char* xs = lds + (s & 1) * kGemmStage;
    const unsigned char* ys = xs + 2 * kGemmStage;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      bf16x8 fx[8], fy[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) fy[b] = staged_frag<YKR>(ys, 64 * wy + 16 * b, kb, t.g, t.i);
#pragma unroll
      for (int a = 0; a < 8; ++a) fx[a] = staged_frag<XKR>(xs, 128 * wx + 16 * a, kb, t.g, t.i);
#pragma unroll
      for (int a = 0; a < 8; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] = pgn_mfma(fx[a], fy[b], acc[a][b]);
    }
  }
  // the buffers may be written again
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Tile `item` of a grid of tx x ty tiles (x tiles, y tiles), so ordered that consecutive items share operands: bands of
// eight y tiles, within a band y fastest.
PGN_DEVICE void band_tile(int64_t item, int64_t tx, int64_t ty, int64_t& ix, int64_t& iy) {
  constexpr int64_t kBand = 8;
  const int64_t band = item / (tx * kBand), y0 = band * kBand, h = min(kBand, ty - y0), in = item - band * tx * kBand;
  ix = in / h;
  iy = y0 + in - ix * h;
}

// The item of workgroup `wg` of `items`, the grid rounded up to a multiple of the XCD count: workgroup wg runs on XCD
// wg % 8, which takes a contiguous run of the items, so neighbours share operands in its L2. -1: none.
PGN_DEVICE int64_t xcd_item(int64_t wg, int64_t items) {
  const int64_t per = (items + kXcdCount - 1) / kXcdCount, item = (wg % kXcdCount) * per + wg / kXcdCount;
  return item < items && wg / kXcdCount < per ? item : -1;
}

inline unsigned xcd_grid(int64_t items) {
  return (unsigned)((items + kXcdCount - 1) / kXcdCount * kXcdCount);
}

}  // namespace pgn
