// ready.hpp — what the activations' preparation leaves in memory for 4 quantized values a lane (quantize.hip's
// ready_kernel and norm.hip).
#pragma once
#include "common.hpp"

namespace hq {

// The 4 bytes of `o` (the lane's values at .. at + 3 of the token; 8 lanes a group of 32, 16 a block of 64, at a multiple of
// 4 times the lane in its wave) to the token's bytes `to` and scales `st`, and per MODE interleave()'s planes and negated
// group sums (1: ternary, binary; n a multiple of 64) or sums_x's int16 sums of 16 and 8 (2: llama.cpp's blocks).  Every lane
// of a wave calls it; a lane that is not `live` stores nothing.
template <int MODE>
HQ_DEV void store_ready(const Quantized4 &o, char *to, char *st, int at, int32_t n, int lane, bool live) {
  const int g = at >> 5;
  if (live && (lane & 7) == 0) ((float *)st)[g] = o.scale;
  if (MODE == 0) {
    if (live) *(uint32_t *)(to + at) = o.d;
    return;
  }
  if (MODE == 1) {
    const int32_t s32 = o.s16 + dpp<0x141>(o.s16);
    if (live && (lane & 7) == 0) ((int32_t *)st)[(n >> 5) + g] = -s32;
    // byte 16 p + c of a block of 64 is value 4 c + p: the quad m of the block's 16 lanes holds c = 4 m .. + 3, and
    // its lane p gathers byte p of the four lanes into the dword at 16 p + 4 m
    const uint32_t q0 = (uint32_t)dpp<0x00>((int32_t)o.d), q1 = (uint32_t)dpp<0x55>((int32_t)o.d);
    const uint32_t q2 = (uint32_t)dpp<0xAA>((int32_t)o.d), q3 = (uint32_t)dpp<0xFF>((int32_t)o.d);
    const uint32_t p = lane & 3, sel = p | ((4 + p) << 8);
    const uint32_t plane = perm(perm(q3, q2, sel), perm(q1, q0, sel), 0x05040100u);
    if (live) *(uint32_t *)(to + (at & ~63) + 16 * p + (lane & 12)) = plane;
  } else {
    int16_t *a16 = (int16_t *)(st + 4 * (n >> 5)), *a8 = a16 + (n >> 4);
    if (live) {
      *(uint32_t *)(to + at) = o.d;
      if ((lane & 1) == 0) a8[at >> 3] = (int16_t)o.s8;
      if ((lane & 3) == 0) a16[at >> 4] = (int16_t)o.s16;
    }
  }
}

}  // namespace hq
