// Activations in 8 bits (rows8.hip): what a layer keeps of its input between
// the forward and the backward.
//   codes [ceil(B / 4)][ld] uint32: byte v of word (t, i) is the code of
//         sample 4 t + v, input i (0 past the batch and past the row);
//   rows  [B][2] float: a sample's offset lo and step; a code stands for
//         lo + code * step.
#pragma once
#include "slg_common.h"

namespace slg {

constexpr int kRows8Tile = 4;  // samples a word

// Words from one tile's row to the next: whole quads, so that every row
// starts at a multiple of 16 bytes.
inline int64_t rows8_ld(int64_t D) { return (D + 3) & ~int64_t(3); }

}  // namespace slg
