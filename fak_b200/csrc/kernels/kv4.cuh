// Layout of the 4-bit KV cache and the small PTX wrappers its kernels share.
//
// One (page of 16 tokens, KV head) is one contiguous block of 20 D bytes (2560 at head dim 128, 1280
// at 64), so a page streams with one bulk copy.  Groups of 32 dims (NG = D / 32) share a scale and a
// minimum; a value is code * scale + minimum, code in [0, 15]:
//   K codes   [16 tokens][4 t][NG groups] u32       dim = group * 32 + t * 8 + nibble (lowest first)
//   K scales  [16 tokens][NG] f16, K minima the same
//   V codes   [8 token pairs][8 x][NG][2 tokens] u16 dim = group * 32 + g * 4 + nibble, g = x ^ 2 (pair & 3)
//   V scales  [8 token pairs][NG][2 tokens] f16, V minima the same
// The orders are those in which a warp's m16n8k16 fragments want them: lane (g, t) reads 16 contiguous
// bytes of K for its token (all groups of its dims) and 16 of V for its token pair, and one AND turns a
// word into a half2 of codes.  The XOR in x keeps the V reads of a warp on distinct banks.
#pragma once
#include "common.cuh"

namespace fak {
namespace kv4 {

constexpr int PAGE = 16;

template <int D>
struct Lay {
  static constexpr int NG = D / 32;
  static constexpr int KC = 0;
  static constexpr int KS = 8 * D;
  static constexpr int KM = KS + 32 * NG;
  static constexpr int VC = KM + 32 * NG;
  static constexpr int VS = VC + 8 * D;
  static constexpr int VM = VS + 32 * NG;
  static constexpr int BYTES = VM + 32 * NG;
  // byte of the u16 that holds dims group * 32 + 4 j .. + 3 of token tok
  FAK_DEV static int k_u16(int tok, int grp, int j) { return KC + tok * (D / 2) + ((j >> 1) * NG + grp) * 4 + (j & 1) * 2; }
  FAK_DEV static int v_u16(int tok, int grp, int j) {
    const int p = tok >> 1;
    return VC + ((p * 8 + (j ^ (2 * (p & 3)))) * NG + grp) * 4 + (tok & 1) * 2;
  }
  FAK_DEV static int k_meta(int tok, int grp) { return (tok * NG + grp) * 2; }                             // from KS / KM
  FAK_DEV static int v_meta(int tok, int grp) { return (((tok >> 1) * NG + grp) * 2 + (tok & 1)) * 2; }    // from VS / VM
};
static_assert(Lay<128>::BYTES == 2560 && Lay<64>::BYTES == 1280, "page bytes");

}  // namespace kv4
}  // namespace fak
