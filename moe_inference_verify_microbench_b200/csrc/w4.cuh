// Expert weights in 4 bits with a scale (and optionally a zero point) for each
// group of `group` consecutive columns of a row:
//   w[n, c] = s[n, c / group] * (q[n, c] - z[n, c / group]),  q, z in 0..15
// (z = 8 where no zero points are kept), s in bf16, group 32, 64 or 128.
//
// Packed layout, written once when the weights are loaded (w4_pack):
//   q  [expert][tile][block][32 lanes][16 bytes]  tile: 16 rows, block: 64 columns
//   s  [expert][tile][group][8][2] bf16           the scales of rows g and g + 8
//   z  [expert][tile][group][8][2] uint8          their zero points
// Lane 4g + t of a block holds rows g and g + 8 of the tile, columns 8t..8t+7 and
// 32 + 8t..32 + 8t+7: {row g first, row g second, row g+8 first, row g+8 second},
// eight codes to a word.  Within a word, nibble i holds column 2i and nibble
// i + 4 column 2i + 1 (i < 4), so (w >> 4i) & 0x000f000f is the column pair in
// the halves of a register: the operand order of mma.m16n8k16, whose K order is
// free as long as both operands agree.  A tile of the gate/up projections is 8
// gate rows followed by the 8 up rows of the same indices, so one thread ends
// up with both and applies the SwiGLU without an exchange.
#pragma once

#include "ptx.cuh"

namespace moe {

constexpr int kW4BlockBytes = 512;  // 16 rows x 64 columns

// One packed projection of every expert.
struct W4Matrix {
  const uint8_t* q;
  const uint8_t* s;  // bf16
  const uint8_t* z;  // null: 8 throughout
  int tiles;         // 16-row tiles per expert
  int nb;            // 64-column blocks per tile
  int ng;            // groups per row
  int gshift;        // log2(group / 32)
};

// The codes of one word's column pair i as bf16 pairs 128 + q: 0x4300 is
// 128.0 and a code is the last four bits of the seven-bit mantissa, so the or
// is exact.
__device__ __forceinline__ uint32_t w4_pair(uint32_t w, int i) {
  return ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
}

// bf16 pair a - b, exact for the small integers used here.
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                   *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// d = a * b + c, 16 x 8 x 16, bf16 operands, fp32 accumulate.
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
        "f"(c[2]), "f"(c[3]));
}

// How a projection is cut over a CTA's eight consumer warps (w4_plan):
// `ks` warps share a tile, `kbn` blocks of 64 columns each, and tl = 8 / ks
// tiles are worked on at once; a ring stage holds `ts` whole tiles of one
// expert with their scales and zero points.
struct W4Plan {
  int ks, tl, kbn;
  int ts;          // tiles per stage
  int groups;      // stages' worth of tiles per expert
  int nr;          // records that share one pass over the weights
  int stages;
  int s_off, z_off, stage_bytes;
};

constexpr int kW4Warps = 8;
// Two consumer warpgroups and a third whose first thread produces.  The block
// launches with 168 registers a thread; the consumers then take 232 and the
// third group keeps 40: 2 * 128 * 232 + 128 * 40 = 384 * 168.
constexpr int kW4Threads = 32 * (kW4Warps + 4);
constexpr int kW4ConsumerRegs = 232;
constexpr int kW4ProducerRegs = 40;
static_assert(32 * kW4Warps * kW4ConsumerRegs + 128 * kW4ProducerRegs <= kW4Threads * 168,
              "the register split must fit what the block launches with");
constexpr int kW4MaxStages = 16;

}  // namespace moe
