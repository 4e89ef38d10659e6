// Table dequantisation of packed nuq codes, shared by the kernels that read the pool.
#pragma once

#include "common.cuh"

namespace hx {

// LUT dequant helpers. A table of 2-byte levels sits 256-aligned in smem; the
// element's byte (2 * code, with the lane's table-offset low bits OR-ed in)
// replaces the low byte of the table's base address in one prmt, and the
// load carries the per-channel offset as its immediate.
HX_DEVINL uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
HX_DEVINL uint16_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
// 8 levels for 8 consecutive 4-bit codes of word w (channels c0 .. c0+7):
// tab(c) = base + off + TSTRIDE * (c - c0). Only base's low byte is replaced,
// so off (a multiple of the table span, folded into the load's immediate once
// unrolled) must be added after the prmt.
template <int TSTRIDE>
HX_DEVINL uint4 lut8_nib(uint32_t w, uint32_t lowbits, uint32_t base, uint32_t off) {
  const uint32_t lo = ((w << 1) & 0x1E1E1E1Eu) | lowbits;  // 2 * code of nibbles 0, 2, 4, 6
  const uint32_t hi = ((w >> 3) & 0x1E1E1E1Eu) | lowbits;  // nibbles 1, 3, 5, 7
  uint16_t v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = lds16(prmt(lo, base, 0x7650u | k) + off + TSTRIDE * (2 * k));
    v[2 * k + 1] = lds16(prmt(hi, base, 0x7650u | k) + off + TSTRIDE * (2 * k + 1));
  }
  return make_uint4(pack_u16x2(v[0], v[1]), pack_u16x2(v[2], v[3]), pack_u16x2(v[4], v[5]),
                    pack_u16x2(v[6], v[7]));
}

// 8 levels for 8 consecutive 4-bit codes of word w from a 16-entry table held
// in registers as byte planes: lb[k] = the low bytes of levels 4k .. 4k+3, hb[k]
// the high bytes. prmt picks a byte out of 8 by a selector nibble's low three
// bits (bit 3, the sign-replicate flag, is cleared), so each plane half gives
// levels code & 7 and 8 + (code & 7); a second prmt takes byte i from the first
// or the second result by code bit 3, and a third interleaves low and high
// bytes into fp16 pairs. No shared-memory access.
HX_DEVINL uint4 lut8_reg(uint32_t w, const uint32_t (&lb)[4], const uint32_t (&hb)[4]) {
  const uint32_t s = w & 0x77777777u;                  // nibble i: code_i & 7
  const uint32_t t = ((w >> 1) & 0x44444444u) | 0x32103210u;  // nibble i: (i & 3) + 4 (code_i >> 3)
  const uint32_t sh = s >> 16, th = t >> 16;
  const uint32_t lo0 = prmt(prmt(lb[0], lb[1], s), prmt(lb[2], lb[3], s), t);    // low bytes, codes 0..3
  const uint32_t hi0 = prmt(prmt(hb[0], hb[1], s), prmt(hb[2], hb[3], s), t);    // high bytes, codes 0..3
  const uint32_t lo1 = prmt(prmt(lb[0], lb[1], sh), prmt(lb[2], lb[3], sh), th);  // codes 4..7
  const uint32_t hi1 = prmt(prmt(hb[0], hb[1], sh), prmt(hb[2], hb[3], sh), th);
  return make_uint4(prmt(lo0, hi0, 0x5140u), prmt(lo0, hi0, 0x7362u), prmt(lo1, hi1, 0x5140u),
                    prmt(lo1, hi1, 0x7362u));
}

HX_DEVINL void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
}
HX_DEVINL uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// 16 levels for 16 consecutive 2-bit codes of word w from level-pair tables:
// a nibble (two codes) picks one 4-byte entry holding both levels, so each
// load yields two channels. tab(pair n) = base + off + TSTRIDE * n, entry
// 4 * nibble; as in lut8_nib only base's low byte is replaced.
template <int TSTRIDE>
HX_DEVINL void lut8_pair(uint32_t w, uint32_t lowbits, uint32_t base, uint32_t off, uint4& o0, uint4& o1) {
  const uint32_t lo = ((w << 2) & 0x3C3C3C3Cu) | lowbits;  // 4 * low nibble: codes 4k, 4k+1
  const uint32_t hi = ((w >> 2) & 0x3C3C3C3Cu) | lowbits;  // 4 * high nibble: codes 4k+2, 4k+3
  uint32_t v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = lds32(prmt(lo, base, 0x7650u | k) + off + TSTRIDE * (2 * k));
    v[2 * k + 1] = lds32(prmt(hi, base, 0x7650u | k) + off + TSTRIDE * (2 * k + 1));
  }
  o0 = make_uint4(v[0], v[1], v[2], v[3]);
  o1 = make_uint4(v[4], v[5], v[6], v[7]);
}

// 16 levels for 16 consecutive 2-bit codes of word w, as two 8-wide chunks.
template <int TSTRIDE>
HX_DEVINL void lut16_crumb(uint32_t w, uint32_t lowbits, uint32_t base, uint32_t off, uint4& o0,
                           uint4& o1) {
  uint32_t g[4];
  g[0] = ((w << 1) & 0x06060606u) | lowbits;  // crumbs 0, 4, 8, 12
  g[1] = ((w >> 1) & 0x06060606u) | lowbits;  // crumbs 1, 5, 9, 13
  g[2] = ((w >> 3) & 0x06060606u) | lowbits;  // crumbs 2, 6, 10, 14
  g[3] = ((w >> 5) & 0x06060606u) | lowbits;  // crumbs 3, 7, 11, 15
  uint16_t v[16];
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int sft = 0; sft < 4; ++sft)
      v[4 * k + sft] = lds16(prmt(g[sft], base, 0x7650u | k) + off + TSTRIDE * (4 * k + sft));
  o0 = make_uint4(pack_u16x2(v[0], v[1]), pack_u16x2(v[2], v[3]), pack_u16x2(v[4], v[5]), pack_u16x2(v[6], v[7]));
  o1 = make_uint4(pack_u16x2(v[8], v[9]), pack_u16x2(v[10], v[11]), pack_u16x2(v[12], v[13]),
                  pack_u16x2(v[14], v[15]));
}

}  // namespace hx
