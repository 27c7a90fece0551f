// The 4-bit paged KV cache.  A layer is two tensors,
//   codes  uint8 [P, 2, Hkv, PS, D/2]      K (0) and V (1) rows of D 4-bit codes
//   scales bf16  [P, 2, Hkv, PS, D/64, 2]  one (scale s, offset z) pair per group of 64 elements
// and element x of a row stands for s * c + z.  A group with least element a
// and largest b has s = bf16((b - a) r) with r the fp32 number next to 1/15 (a
// product costs less than a division and differs from it in the last fp32 bit at
// most, so s only where the quotient lies that near to a border between two bf16
// numbers), z = bf16(a) and
// c = round((x - z) / s) clamped to 0..15 (0 where s is 0); a group that holds
// a NaN or an infinity gets s = z = NaN, so every element of it reads as NaN.
// A row of 128 elements takes 64 + 8 bytes instead of 256.
//
// Order within a row: D / 8 little-endian 32-bit words of 8 codes; word
// 2 i + h holds elements 8 i + h D/2 .. + 7, element j in bits 4 j .. 4 j + 3.
// Interleaving the two halves of a row lets one 8- or 16-byte load give a
// thread words of both groups (D 128) and both members of a rotary pair.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "common.cuh"

namespace braid {

constexpr int KV4_GROUP = 64;

// Place of logical word l (elements 8 l .. 8 l + 7) within its row.
template <int D>
BRAID_DEVICE int kv4_word(int l) {
  constexpr int HALF = D / 16;
  return 2 * (l % HALF) + l / HALF;
}

BRAID_DEVICE float kv4_scale(uint32_t sz) { return __uint_as_float(sz << 16); }
BRAID_DEVICE float kv4_offset(uint32_t sz) { return __uint_as_float(sz & 0xFFFF0000u); }

}  // namespace braid
