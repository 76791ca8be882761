// Expert weights in 4 bits with a scale (and optionally a zero point) for each
// group of `group` consecutive columns of a row:
//   w[n, c] = s[n, c / group] * (q[n, c] - z[n, c / group]),  q, z in 0..15
// (z = 8 where no zero points are kept), s in bf16, group 32, 64 or 128.
//
// Packed layout, written once when the weights are loaded (w4_pack):
//   q  [expert][tile][block][32 lanes][16 bytes]  tile: 16 rows, block: 64 columns
//   s  [expert][tile][group][8] records of rows g and g + 8: two bf16 scales and,
//      with zero points, two bf16 values 128 + z
// Lane 4g + t of a block holds rows g and g + 8 of the tile: {row g columns 0..31,
// row g 32..63, row g+8 0..31, row g+8 32..63}, eight codes to a word.  Within a
// word, nibble i holds column 8i + 2t and nibble i + 4 column 8i + 2t + 1 (i < 4)
// of the word's 32, so (w >> 4i) & 0x000f000f is a column pair in the halves of a
// register: the fragment order of a 16-row matrix operand, both for mma.m16n8k16
// and for tcgen05.st.16x128b into tensor memory.  A tile of the gate/up
// projections is 8 gate rows followed by the 8 up rows of the same indices, so
// one thread ends up with both and applies the SwiGLU without an exchange.
#pragma once

#include <atomic>

#include "internal.h"
#include "ptx.cuh"

namespace moe {

constexpr int kW4BlockBytes = 512;  // 16 rows x 64 columns

// One packed projection of every expert.
struct W4Matrix {
  const uint8_t* q;
  const uint8_t* s;
  int rec;           // bytes of a record: 4, or 8 with zero points
  int tiles;         // 16-row tiles per expert
  int nb;            // 64-column blocks per tile
  int ng;            // groups per row
  int gshift;        // log2(group / 32)
};

// The column pairs of a word as bf16 pairs 128 + q: 0x4300 is 128.0 and a code is
// the last four bits of the seven-bit mantissa, so the or is exact: seven integer
// instructions for eight codes.
template <uint32_t BASE = 0x43004300u>
__device__ __forceinline__ void w4_pairs(uint32_t w, uint32_t (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("lop3.b32 %0, %1, %2, %3, 0xea;"
        : "=r"(r[i])
        : "r"(w >> (4 * i)), "n"(0x000f000f), "r"(BASE));
}

// bf16 pair a - b, exact for the small integers used here.
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// d += a * b, 16 x 8 x 16, bf16 operands, fp32 accumulate.
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// How a projection is cut over a CTA's sixteen warps (w4_plan): `ks` warps share
// a tile, kb blocks of 64 columns each (a kernel parameter; blocks past the last
// are multiplied with zeros), and tl = 16 / ks such groups work side by side.
struct W4Plan {
  int ks, tl;
  int ks_shift;            // log2(ks)
  int slot_bytes;          // one tile's share of a warp: codes, then records
};

// How often a warp applies scales: after every two blocks, after every block, or
// after every 32 columns.  The last also subtracts zero points from each operand.
enum W4Mode : int { kW4TwoBlocks = 0, kW4Block = 1, kW4Half = 2 };
constexpr int kW4Recs = 8;  // records that share one pass over the weights

constexpr int kW4Warps = 16;
constexpr int kW4Threads = 32 * kW4Warps;

// Operands of a grouped product with 4-bit weights.
struct W4Args {
  W4Matrix m;
  W4Plan p;
  const uint32_t* act;  // A rows [act_rows][K], bf16 pairs
  int act_rows;
  const int* index;     // A row of record p = act[index[p] / index_div] (null = p)
  int index_div;
  int M;                // records
  const int4* tiles;
  const int* num_tiles;
  int max_tiles;
  int E;
  __nv_bfloat16* out;
  float* out_f32;       // where the rows go instead, unrounded (the stream's down product and
                        // the tensor-memory form's gate/up product)
  const float* row_factor;  // tensor-memory form: of the weight rows [expert][tile][16], of
                            // the experts behind them
  const float* act_factor;  // and of the A rows
  int out_ld;
  int out_rows;
  const int* row_map;
  const float* row_scale;
  bool zero_rest;       // rows of out before the first entry and after the last are zeroed
  int* status;
};

// `threads` threads (whole warps) meet at barrier `id`.  bar.sync wants a converged
// warp, and lanes may come from a branch.
__device__ __forceinline__ void named_barrier(int id, int threads) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}

__device__ __forceinline__ void lds64(uint32_t addr, uint32_t& x, uint32_t& y) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(addr));
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// Whether a tile-table entry is an expert's row range of at most kBM rows; a bad one is
// reported (an empty one is not) and skipped.
__device__ __forceinline__ bool w4_entry_ok(const W4Args& a, const int4& t) {
  if (t.x >= 0 && t.x < a.E && t.y >= 0 && t.y < t.z && t.z <= a.M && t.z - t.y <= 128) return true;
  if (t.x < 0 || t.x >= a.E) record_status(a.status, kErrBadExpert);
  else if (t.y != t.z) record_status(a.status, kErrBadRow);
  return false;
}

// Zeroes the output rows before the first of nt entries and after the last (all rows,
// where there are none), with `count` threads of every CTA.
__device__ __forceinline__ void w4_zero_rest(const W4Args& a, int nt, int thread, int count) {
  if (!a.zero_rest) return;
  const int first = nt > 0 ? max(0, min(a.tiles[0].y, a.out_rows)) : a.out_rows;
  const int last = nt > 0 ? max(first, a.tiles[nt - 1].z) : a.out_rows;
  const int vec = a.out_ld / 8;
  for (long long i = blockIdx.x;; i += gridDim.x) {
    const long long r = i < first ? i : last + (i - first);
    if (r >= a.out_rows) break;
    uint4* row = reinterpret_cast<uint4*>(a.out + static_cast<size_t>(r) * a.out_ld);
    for (int v = thread; v < vec; v += count) row[v] = make_uint4(0, 0, 0, 0);
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class Kernel>
bool allow_smem(Kernel* fn, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if ((done.load(std::memory_order_acquire) & bit) != 0) return true;
  if (note_cuda_error(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           bytes)) != cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_acq_rel);
  return true;
}

// The tensor-memory form for experts with many records (w4_gemm.cu), from
// kW4TcRecords records per expert on.  f32: a.act holds fp32 rows, which it overwrites.
int w4_gemm(W4Args a, bool swiglu, const W4Rows& rows, bool f32, cudaStream_t stream);

}  // namespace moe
