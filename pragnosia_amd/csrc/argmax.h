// The largest of many values and its index, by ordered keys and lane moves in the vector unit (decode_tail, rules).
#pragma once
#include "common.h"

namespace {

// A logit as an unsigned number in torch.argmax's order: NaN (any) above every number, -0 equal to +0. Above 0 always.
PGN_DEVICE unsigned order_key(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  if (x != x) return 0xffffffffu;
  if (u == 0x80000000u) return 0x80000000u;  // -0 as +0
  return u >> 31 ? ~u : u | 0x80000000u;
}

// (order key, ~index) as one 64-bit number: the larger is the better logit, the smaller index among equals
struct Key {
  unsigned hi, lo;
};
PGN_DEVICE Key max_key(const Key& a, const Key& b) {
  return a.hi > b.hi || (a.hi == b.hi && a.lo > b.lo) ? a : b;
}
template <int CTRL>
PGN_DEVICE Key max_dpp(const Key& k) {
  return max_key(k, Key{(unsigned)__builtin_amdgcn_update_dpp(0, (int)k.hi, CTRL, 0xf, 0xf, true),
                        (unsigned)__builtin_amdgcn_update_dpp(0, (int)k.lo, CTRL, 0xf, 0xf, true)});
}
// Over each row of 16 lanes, in all of them (group_sum's exchanges)
PGN_DEVICE Key max_row(Key k) {
  k = max_dpp<0xB1>(k);    // quad_perm [1, 0, 3, 2]
  k = max_dpp<0x4E>(k);    // quad_perm [2, 3, 0, 1]
  k = max_dpp<0x141>(k);   // row_half_mirror
  return max_dpp<0x140>(k);  // row_mirror
}
// Over the wave's 64 lanes, in all of them: a swap of a register with itself leaves the two halves' values side by side
PGN_DEVICE Key max_wave(Key k) {
  k = max_row(k);
  {
    const auto h = __builtin_amdgcn_permlane16_swap(k.hi, k.hi, false, false);
    const auto l = __builtin_amdgcn_permlane16_swap(k.lo, k.lo, false, false);
    k = max_key(Key{h[0], l[0]}, Key{h[1], l[1]});
  }
  const auto h = __builtin_amdgcn_permlane32_swap(k.hi, k.hi, false, false);
  const auto l = __builtin_amdgcn_permlane32_swap(k.lo, k.lo, false, false);
  return max_key(Key{h[0], l[0]}, Key{h[1], l[1]});
}

}  // namespace
