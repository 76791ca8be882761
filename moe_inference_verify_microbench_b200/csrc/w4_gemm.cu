// Grouped products with 4-bit expert weights on tcgen05, for experts with many
// records (layout: w4.cuh; the form for few records: w4.cu).
//
// The weights are the 128-row operand and live in tensor memory: sixteen warps turn
// codes into fp16 s * (q - z) in registers, in the fragment order that
// tcgen05.st.16x128b writes, so the dequantised weights never touch shared
// memory, whose bandwidth the operand reads of 128-row tiles would fill.  The
// records are the N operand (16 to 128 columns of one tile-table entry) in
// shared memory, and the accumulators hold D[weight row][record].  So a pass
// over an expert's weights costs the same integer work for 16 records as for
// 128: about 60 instructions per 16 x 64 block (28 to extract, 32 to subtract
// and scale), which bounds small N.
//
// Work unit: (tile-table entry, 16 packed tiles), i.e. 256 weight rows as two
// operands of 128 that share the records: for the gate/up product the gate rows
// and the up rows of the same 128 outputs (the two accumulators then hold gate
// and up in the same lane and column), for the down product two runs of 128 rows.
//
// CTA (864 threads, one per SM, persistent):
//   warps 0..15   dequantise: warp w writes lane quarter w % 4 of every fourth
//                 64-column block
//   warps 16..19  epilogue: tensor memory -> bf16 -> staging rows -> output rows (h that the
//                 down product reads next: fp32, from the registers to its rows)
//   warps 20..23  gather the records' rows (tile::gather4: four rows a copy, into the
//                 128-byte swizzle; one warp for all copies of 128 records was the
//                 bound: 8192 tokens 1578 us instead of 863 then)
//   warp 24       tiled copies of codes and group records into a ring
//   warps 25, 26  issue tcgen05.mma, one operand each: 4 steps of 16 columns per
//                 block; warp 25 allocates tensor memory
//
// Numerics: a weight s * (q - z) has twelve bits, eight of the bf16 scale and four; fp16
// operands round it to eleven, 2^-12 of it at most (bf16 would leave eight: three such
// roundings made the error of the whole call 3.8e-3 of 64 bits, where y and the slot rows
// alone make 2.4e-3).  fp16's range is met by powers of two: an expert's scales are
// multiples of one (w4_pack_fine; much smaller rows of their own), a row of activations of
// another (w4_rows_f16, which also rounds h, fp32 from the gate/up product, to fp16:
// 2^-12).  They come off the fp32 sums in the epilogue, exactly.
//
// Measured, 128 experts of 2048 x 768, group 128, one launch with L2 cold, gate/up and
// down: 16 records per expert 70 and 38 us (3.0 and 2.7 TB/s of codes), 512 records 498
// and 289 us (0.83 and 0.71 PFLOP/s); with bf16 operands and h they took 67, 38, 470 and 286.
// Activations to fp16: 8192 x 2048 bf16 10 us, 65536 x 768 fp32 41 us (HBM), small ones 4.
// At 16 records the issue slots are three quarters used (66 instructions per 16 x 64
// block of codes for the dequantisation, about 30 for all else) and a set of warps waits
// for its own products before it refills its stage; a third pair of stages was worth 3 %.
// Halves of units in a last round that is not half full cost as much as whole ones (shard
// of 32 experts 78 -> 84 us).  At 512 the tiles of 128 records and 256 weight rows move 6
// TB/s from L2, and their products wait for the epilogue before them (5000 of 34000
// cycles for gate/up), because tensor memory holds 128 records' sums once.
#include <algorithm>

#include "grouped_gemm.cuh"
#include "w4.cuh"

namespace moe {

namespace {

constexpr int kTcStages = 4;      // weight operand stages (64 columns) in tensor memory
constexpr int kTcPairs = 2;       // of them that are handed over together
// Record slots in shared memory (see tc_blocks).
template <bool SWIGLU>
constexpr int kTcSlots = SWIGLU ? 6 : 4;
constexpr int kTcRing = 4;        // code stages (128 columns)
constexpr int kTcTiles = 16;      // packed tiles per unit
constexpr int kTcBlocks = 2;      // blocks per code stage
constexpr int kTcRows = 128;      // records per unit at most
constexpr int kTcDequantWarps = 16;
constexpr int kTcEpiWarp = 16, kTcLoadWarp = 20, kTcCopyWarp = 24, kTcMmaWarp = 25;
constexpr int kTcLoadWarps = kTcCopyWarp - kTcLoadWarp;
constexpr int kTcThreads = 27 * 32;
constexpr int kTcBBytes = kTcRows * 128;
// Staging: the outputs of a unit for 128 records, rows 16 bytes apart in banks.  The down
// product has 256 of them, so that its accumulators are free before anything is stored.
template <bool SWIGLU>
constexpr int kTcOutRow = (SWIGLU ? 256 : 512) + 16;
constexpr int kTcCodeBytes = kTcTiles * kTcBlocks * kW4BlockBytes;
constexpr uint32_t kTcOperandCol = 256;     // accumulators below, operand stages above

struct TcArgs {
  W4Args a;
  int ring_bytes;  // code stage: codes, then records
  int rec_stride;  // bytes of a tile's records in it
};

__device__ __forceinline__ void tmem_st_16x128b_x8(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

// 32 lanes, 16 columns from taddr on, a row to a lane.
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

// 16 lanes, 16 columns from taddr on, in the order of product fragments: lane
// 4 g + t has columns 2t, 2t + 1 of rows g and g + 8, then columns 8 + 2t, 9 + 2t.
__device__ __forceinline__ void tmem_ld_16x256b_x2(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr));
}

// Four 8 x 8 blocks of 16-bit values, transposed: lane i names row i % 8 of block i / 8.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile(
      "stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T, fp16 inputs, fp32 accumulate.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t desc_lo,
                                               uint32_t desc_hi, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 bd;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 bd, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], bd, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(desc_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p;
}

// Rows r0..r3, 64 columns from x on, of a tensor map whose box is one row.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* m, uint64_t* bar,
                                            int x, int r0, int r1, int r2, int r3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(r0), "r"(r1), "r"(r2),
      "r"(r3)
      : "memory");
}

// The column pairs of a word as fp16 s * (q - z): 0x6400 is 1024.0 and a code is
// the last four bits of the mantissa; 1024 + q - (1024 + z) is exact, the product
// is rounded once.
__device__ __forceinline__ void w4_scaled_pairs(uint32_t w, uint32_t z, uint32_t s, uint32_t* r,
                                                int stride) {
  uint32_t v[4];
  w4_pairs<0x64006400u>(w, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t d;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(d) : "r"(v[i]), "r"(z));
    asm("mul.f16x2 %0, %1, %2;" : "=r"(r[i * stride]) : "r"(d), "r"(s));
  }
}

// Which accumulator columns a unit uses.  Up to 64 records: one of two halves of
// 128 columns in turn, so that the epilogue of a unit overlaps the next unit's
// products; more: all 256.
struct TcAcc {
  uint32_t used[2] = {0, 0}, filled[2] = {0, 0};
  int next = 0;
  int first, last;     // halves of the current unit
  uint32_t d0, d1;     // its columns
  __device__ __forceinline__ void take(int n) {
    const bool small = n <= 64;
    first = small ? next : 0;
    last = small ? next : 1;
    next = small ? next ^ 1 : 0;
    d0 = first * 128;
    d1 = d0 + (small ? 64 : 128);
  }
};

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Accumulator rows of this warp's lanes times `factor` of the lane's row: for weight rows
// that have a power of two of their own, or an expert whose scales are all below 2^-26 or
// reach 2^24, which are rare.  (The same products in
// the loop that takes the accumulators out cost it 15 % where there are none.)
__device__ __noinline__ void tc_rescale(uint32_t taddr, int cols, float factor) {
  for (int c = 0; c < cols; c += 16) {
    uint32_t v[16];
    tmem_ld16(taddr + c, v);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * factor);
    tmem_st_32x32b_x16(taddr + c, v);
  }
  tmem_wait_st();
}

// Units of the grid in turn: entry, 16-tile group, and whether there is work.
struct TcUnit {
  int4 t;
  int m;
  bool ok;
};
// A record slot is 128 rows of 64 columns; with fewer records it holds as many
// 64-column blocks as fit, so that the same bytes are in flight.
__device__ __forceinline__ int tc_blocks(int n) { return 8 / ((n + 15) >> 4); }

__device__ __forceinline__ TcUnit tc_unit(const W4Args& a, int w, int groups) {
  TcUnit u;
  const int e = w / groups;
  u.m = w - e * groups;
  u.t = a.tiles[e];
  u.ok = w4_entry_ok(a, u.t);
  return u;
}

// Low word of the descriptor of a record block in shared memory.
__device__ __forceinline__ uint32_t tc_desc(uint32_t addr) {
  return ((addr >> 4) & 0x3fffu) | (1u << 16);
}

// Barrier calls by shared-memory address, for the loops that count instructions.
// (Suspending a waiting warp for up to 10 us at a time measured 1 to 2 % slower here.)
__device__ __forceinline__ bool tc_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ void tc_spin(uint32_t bar, uint32_t parity, volatile int* abort,
                                     int* status, int code) {
  const unsigned long long t0 = globaltimer_ns();
  for (uint32_t it = 1; !tc_try(bar, parity); ++it) {
    if ((it & 63u) != 0) continue;
    if (*abort) return;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      record_status(status, code);
      *abort = 1;
      return;
    }
  }
}
__device__ __forceinline__ void tc_wait(uint32_t bar, uint32_t parity, volatile int* abort,
                                        int* status, int code) {
  if (!tc_try(bar, parity)) tc_spin(bar, parity, abort, status, code);
}
__device__ __forceinline__ void tc_commit32(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void tc_arrive32(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// The products of a 64-column block with one operand: four steps of 16 columns.
__device__ __forceinline__ void tc_block(uint32_t d, uint32_t at, uint32_t lo, uint32_t hi,
                                         uint32_t idesc, bool add) {
#pragma unroll
  for (int kk = 0; kk < 4; ++kk)
    tc_mma_f16_ts(d, at + kk * 8, lo + 2 * kk, hi, idesc, kk != 0 || add ? 1u : 0u);
}

// HALVES: groups of 32, two to a block; ZEROS: zero points are kept.
template <bool SWIGLU, bool HALVES, bool ZEROS>
__global__ void __launch_bounds__(kTcThreads, 1)
    w4_tc(const __grid_constant__ CUtensorMap tm_codes,
          const __grid_constant__ CUtensorMap tm_records,
          const __grid_constant__ CUtensorMap tm_rows, const TcArgs args) {
  constexpr int kRec = ZEROS ? 8 : 4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const W4Args& a = args.a;
  uint8_t* sB = smem;
  constexpr int kSlots = kTcSlots<SWIGLU>, kOutRow = kTcOutRow<SWIGLU>;
  uint8_t* sOut = sB + kSlots * kTcBBytes;
  uint8_t* sRing = sOut + kTcRows * kOutRow;
  uint64_t* full = reinterpret_cast<uint64_t*>(sRing + kTcRing * args.ring_bytes);
  uint64_t* empty = full + kTcPairs;
  uint64_t* bfull = empty + kTcPairs;
  uint64_t* bempty = bfull + kSlots;
  uint64_t* qfull = bempty + kSlots;
  uint64_t* qempty = qfull + kTcRing;
  uint64_t* acc_full = qempty + kTcRing;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* store_stop = reinterpret_cast<volatile int*>(tmem_slot + 2);
  float* s_scale = reinterpret_cast<float*>(tmem_slot + 4);
  int* s_row = reinterpret_cast<int*>(s_scale + kTcRows);  // of this unit and of the last one

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kTcPairs; ++s) {
      mbar_init(&full[s], 4 * kTcBlocks);  // the warps of two sets
      mbar_init(&empty[s], 2);  // both issuers'
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bfull[s], kTcLoadWarps);
      mbar_init(&bempty[s], 2);
    }
    for (int s = 0; s < kTcRing; ++s) {
      mbar_init(&qfull[s], 1);
      mbar_init(&qempty[s], 4 * kTcBlocks);  // a set for each block
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 2);
      mbar_init(&acc_empty[b], 4);
    }
    *abort_flag = 0;
    *store_stop = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == kTcMmaWarp) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  const int nt = max(0, min(*a.num_tiles, a.max_tiles));
  const int groups = (a.m.tiles + kTcTiles - 1) / kTcTiles;
  const long long units = static_cast<long long>(nt) * groups;
  const int total = static_cast<int>(min(units, 0x7fffffffLL - static_cast<long long>(gridDim.x)));
  const int nb = a.m.nb;
  const uint32_t nbe = (nb + kTcBlocks - 1) / kTcBlocks * kTcBlocks;

  static_assert(kTcStages == kTcDequantWarps / 4, "an operand stage for each set");

  if (warp < kTcDequantWarps) {
    // ------------------------------------------------------------ dequantise
    // Blocks are counted through all units, an odd number in a unit rounded up to
    // whole code stages; set i of four warps, one per lane quarter, takes the blocks
    // i modulo 4 and fills operand stage i with them.  Two blocks, of sets 0 and 1 or
    // of sets 2 and 3, are handed over together.  So a set's j-th block comes through
    // code stage (set / 2) + 2 (j mod 2).  After an abort the waits return at once and the
    // unit is finished on what the stages hold.
    static_assert(kTcRing == 2 * kTcPairs && kTcBlocks == 2, "the order of a set's stages");
    const int quarter = warp & 3, set = warp >> 2, bk = set & 1;
    const uint32_t dst = tmem + kTcOperandCol + set * 64 + (static_cast<uint32_t>(32 * quarter) << 16);
    const uint32_t stage = smem_u32(sRing) + (set >> 1) * args.ring_bytes;
    const uint32_t q0 = stage + bk * kW4BlockBytes + lane * 16;
    const uint32_t rec0 = stage + kTcCodeBytes + (lane >> 2) * kRec +
                          (HALVES ? 2 * bk : (2 * bk) >> a.m.gshift) * (8 * kRec);
    const uint32_t hand = (set >> 1) * 8;
    const uint32_t qfull0 = smem_u32(qfull) + hand, qempty0 = smem_u32(qempty) + hand,
                   full0 = smem_u32(full) + hand, empty0 = smem_u32(empty) + hand;
    uint32_t base = 0;  // blocks before this unit
    uint32_t j = 0;     // of this set
    for (int w = blockIdx.x; w < total; w += gridDim.x) {
      const TcUnit u = tc_unit(a, w, groups);
      if (!u.ok) continue;
      if (!__all_sync(0xffffffffu, *abort_flag == 0)) break;
      const int left = a.m.tiles - u.m * kTcTiles;  // packed tiles from here to the end
      for (uint32_t kb = (set - base) & 3u; kb < nbe; kb += 4, ++j) {
        const uint32_t odd = j & 1u;
        tc_wait(qfull0 + 16 * odd, (j >> 1) & 1u, abort_flag, a.status, kErrTimeoutFull);
        tc_wait(empty0, odd ^ 1u, abort_flag, a.status, kErrTimeoutEmpty);
        __syncwarp();
        tc_fence_after();
        // none for a block that rounds the unit up
        const int tiles = kb < static_cast<uint32_t>(nb) ? left : 0;
        const uint32_t q = q0 + odd * (2 * args.ring_bytes), rec = rec0 + odd * (2 * args.ring_bytes);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // two packed tiles: 16 gate and 16 up rows, or 32 rows
          const int tile0 = SWIGLU ? 4 * quarter + 2 * half : 8 * half + 2 * quarter;
          if (tile0 < tiles) {
            const uint4 w0 = lds128(q + tile0 * (kTcBlocks * kW4BlockBytes));
            const uint4 w1 = lds128(q + (tile0 + 1) * (kTcBlocks * kW4BlockBytes));
            // [half block] of {tile 0, tile 1} x {row g, row g + 8}
            uint32_t sc[2][2][2], zp[2][2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                if (HALVES || h == 0) {
                  const uint32_t r = rec + (tile0 + i) * args.rec_stride + h * (8 * kRec);
                  uint32_t sv, zv = 0;  // scales of rows g, g + 8, and 1024 + z
                  if (ZEROS) lds64(r, sv, zv);
                  else sv = lds32(r);
                  sc[h][i][0] = __byte_perm(sv, 0, 0x1010);
                  sc[h][i][1] = __byte_perm(sv, 0, 0x3232);
                  zp[h][i][0] = ZEROS ? __byte_perm(zv, 0, 0x1010) : 0x64086408u;
                  zp[h][i][1] = ZEROS ? __byte_perm(zv, 0, 0x3232) : 0x64086408u;
                } else {
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    sc[1][i][k] = sc[0][i][k];
                    zp[1][i][k] = zp[0][i][k];
                  }
                }
              }
            }
            uint32_t r[16];
            if constexpr (SWIGLU) {
              // gate rows of both tiles, then their up rows, as 16 operand rows each
              w4_scaled_pairs(w0.x, zp[0][0][0], sc[0][0][0], r, 2);
              w4_scaled_pairs(w0.y, zp[1][0][0], sc[1][0][0], r + 8, 2);
              w4_scaled_pairs(w1.x, zp[0][1][0], sc[0][1][0], r + 1, 2);
              w4_scaled_pairs(w1.y, zp[1][1][0], sc[1][1][0], r + 9, 2);
              tmem_st_16x128b_x8(dst + (static_cast<uint32_t>(16 * half) << 16), r);
              w4_scaled_pairs(w0.z, zp[0][0][1], sc[0][0][1], r, 2);
              w4_scaled_pairs(w0.w, zp[1][0][1], sc[1][0][1], r + 8, 2);
              w4_scaled_pairs(w1.z, zp[0][1][1], sc[0][1][1], r + 1, 2);
              w4_scaled_pairs(w1.w, zp[1][1][1], sc[1][1][1], r + 9, 2);
              tmem_st_16x128b_x8(dst + 32 + (static_cast<uint32_t>(16 * half) << 16), r);
            } else {
              w4_scaled_pairs(w0.x, zp[0][0][0], sc[0][0][0], r, 2);
              w4_scaled_pairs(w0.y, zp[1][0][0], sc[1][0][0], r + 8, 2);
              w4_scaled_pairs(w0.z, zp[0][0][1], sc[0][0][1], r + 1, 2);
              w4_scaled_pairs(w0.w, zp[1][0][1], sc[1][0][1], r + 9, 2);
              tmem_st_16x128b_x8(dst + 32 * half, r);
              w4_scaled_pairs(w1.x, zp[0][1][0], sc[0][1][0], r, 2);
              w4_scaled_pairs(w1.y, zp[1][1][0], sc[1][1][0], r + 8, 2);
              w4_scaled_pairs(w1.z, zp[0][1][1], sc[0][1][1], r + 1, 2);
              w4_scaled_pairs(w1.w, zp[1][1][1], sc[1][1][1], r + 9, 2);
              tmem_st_16x128b_x8(dst + 32 * half + (16u << 16), r);
            }
          }
        }
        // tcgen05.wait is .sync.aligned: no lane may branch off in front of it
        if ((SWIGLU ? 4 * quarter : 2 * quarter) < tiles) tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          tc_arrive32(qempty0 + 16 * odd);  // the codes have been read
          tc_arrive32(full0);
        }
      }
      base += nbe;
    }
  } else if (warp >= kTcEpiWarp && warp < kTcLoadWarp) {
    // -------------------------------------------------------------- epilogue
    const int quarter = warp & 3;
    const int r = threadIdx.x - kTcEpiWarp * 32;  // record this thread stores
    const uint32_t lanes = static_cast<uint32_t>(32 * quarter) << 16;
    const uint32_t stage = smem_u32(sOut);
    int* rows = s_row;
    if constexpr (!SWIGLU) w4_zero_rest(a, nt, r, 128);
    TcAcc acc;
    bool ok = true;
    for (int w = blockIdx.x; ok && w < total; w += gridDim.x) {
      const TcUnit u = tc_unit(a, w, groups);
      if (!u.ok) continue;
      const int n = u.t.z - u.t.y, cols = (n + 15) & ~15;
      acc.take(cols);
      int o = -1;
      if (r < n) {
        const int p = u.t.y + r;
        o = a.row_map != nullptr ? a.row_map[p] : p;
        if (o < 0 || o >= a.out_rows) {
          record_status(a.status, kErrBadRow);
          o = -1;
        }
      }
      rows[r] = o;
      float scale = !SWIGLU && o >= 0 && a.row_scale != nullptr ? a.row_scale[o] : 1.0f;
      // Times the powers of two of the record's activations (2^-112 to 2^113) and of the
      // expert's scales, unless the two might leave fp32's range together.
      const float base = a.row_factor[static_cast<size_t>(a.E) * a.m.tiles * 16 + u.t.x];
      const bool far = base < 0x1p-36f || base > 0x1p14f;
      if (o >= 0) {
        const int p = u.t.y + r, row = a.index != nullptr ? a.index[p] / a.index_div : p;
        if (row >= 0 && row < a.act_rows) scale *= a.act_factor[row] * (far ? 1.0f : base);
      }
      s_scale[r] = scale;
      const bool wide = SWIGLU && a.out_f32 != nullptr;
      // of this lane's two weight rows, gate and up or one of each operand
      float own[2];
#pragma unroll
      for (int op = 0; op < 2; ++op) {
        const int j = 32 * quarter + lane;
        const int tile = u.m * kTcTiles + (SWIGLU ? j >> 3 : 8 * op + (j >> 4));
        const int row = SWIGLU ? 8 * op + (j & 7) : j & 15;
        const size_t et = static_cast<size_t>(u.t.x) * a.m.tiles + tile;
        own[op] = tile < a.m.tiles ? __ldg(a.row_factor + et * 16 + row) : 1.0f;
        if (far) own[op] *= base;
      }
      const bool rescale = __any_sync(0xffffffffu, own[0] != 1.0f || own[1] != 1.0f);
      ok = mbar_wait_idle(&acc_full[acc.first], acc.filled[acc.first] & 1u, abort_flag, a.status,
                     kErrTimeoutAccFull);
      ok = __all_sync(0xffffffffu, ok);
      ++acc.filled[acc.first];
      tc_fence_after();
      // outputs of this unit from `first`, fewer at the end of the matrix
      constexpr int kOuts = SWIGLU ? 128 : 256;
      const int first = u.m * kOuts;
      const int outs = min(kOuts, a.m.tiles * (SWIGLU ? 8 : 16) - first);
      if (!ok) *store_stop = 1;
      named_barrier(1, 128);
      ok = *store_stop == 0;  // the four warps leave together: they meet at this barrier
      if (rescale && ok) {
        tc_rescale(tmem + lanes + acc.d0, cols, own[0]);
        tc_rescale(tmem + lanes + acc.d1, cols, own[1]);
      }
#pragma unroll
      for (int part = 0; part < kOuts / 128; ++part) {
        if (ok && part * 128 < outs) {
          const uint32_t d = tmem + lanes + (part == 0 ? acc.d0 : acc.d1);
          // records down the staging rows: the fragments go through transposing stores
          const uint32_t dst = stage + ((lane >> 4) * 8 + (lane & 7)) * kOutRow +
                               (128 * part + 32 * quarter + ((lane >> 3) & 1) * 8) * 2;
          // fp32 rows: this lane's first output in its column 2t of the record
          float* to = a.out_f32 + static_cast<size_t>(u.t.y + 2 * (lane & 3)) * a.out_ld + first +
                      32 * quarter + (lane >> 2);
          if (wide && 32 * quarter >= outs) continue;  // outs is a multiple of 64
          for (int c = 0; c < cols; c += 16) {
            uint32_t v[2][8];
            tmem_ld_16x256b_x2(d + c, v[0]);
            tmem_ld_16x256b_x2(d + (16u << 16) + c, v[1]);
            const float* sc = s_scale + c + 2 * (lane & 3);
            const float2 s0 = *reinterpret_cast<const float2*>(sc);
            const float2 s1 = *reinterpret_cast<const float2*>(sc + 8);
            // value i of a fragment: column (i & 1) of 2t, 2t + 1, row g + 8 ((i >> 1) & 1),
            // columns 8 on from i = 4
            auto scaled = [&](uint32_t x, int i) {
              const float2 sv = (i & 4) != 0 ? s1 : s0;
              return __uint_as_float(x) * ((i & 1) != 0 ? sv.y : sv.x);
            };
            if constexpr (SWIGLU) {
              uint32_t up[2][8];
              tmem_ld_16x256b_x2(tmem + lanes + acc.d1 + c, up[0]);
              tmem_ld_16x256b_x2(tmem + lanes + (16u << 16) + acc.d1 + c, up[1]);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                v[i >> 3][i & 7] = __float_as_uint(silu_f(scaled(v[i >> 3][i & 7], i)) *
                                                   scaled(up[i >> 3][i & 7], i));
              if (wide) {
                // straight from the registers: eight lanes write 32 bytes of a record's row
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // columns 2t, 2t + 1, 8 on
                  const int col = (k & 1) + 8 * (k >> 1);
                  if (c + 2 * (lane & 3) + col < n) {
                    float* p = to + col * a.out_ld;
#pragma unroll
                    for (int m = 0; m < 4; ++m)  // rows g, g + 8, 16 on
                      p[8 * m] = __uint_as_float(v[m >> 1][(k & 1) + 2 * (m & 1) + 4 * (k >> 1)]);
                  }
                }
                to += 16 * a.out_ld;
                continue;
              }
            } else {
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                v[i >> 3][i & 7] = __float_as_uint(scaled(v[i >> 3][i & 7], i));
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t pk[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                pk[i] = pack_bf16x2(__uint_as_float(v[h][2 * i]), __uint_as_float(v[h][2 * i + 1]));
              stmatrix_x4_trans(dst + c * kOutRow + h * 32, pk);
            }
          }
        }
      }
      tc_fence_before();  // the accumulators are read
      __syncwarp();
      if (lane == 0) {
        for (int b = acc.first; b <= acc.last; ++b) mbar_arrive(&acc_empty[b]);
      }
      named_barrier(1, 128);
      // Sixteen threads store 128 outputs of a row.  (Bulk copies of whole rows, one from
      // every thread, took 2700 cycles to issue: 16 records per expert 39 us for the down
      // product instead of 36; 512 records 269 instead of 263, but 421 instead of 430 for
      // gate/up, where nobody waits for the stores.)
      constexpr int kPer = kOuts / 8;
      const int v = r % kPer;
      if (ok && v * 8 < outs && !wide) {
        const uint32_t src = stage + v * 16;
        __nv_bfloat16* dst = a.out + first + v * 8;
        for (int c = r / kPer; c < n; c += 4 * (128 / kPer)) {  // four rows in flight
          uint4 val[4];
          int at[4];  // -1 past the last
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = min(c + i * (128 / kPer), kTcRows - 1);
            at[i] = c + i * (128 / kPer) < n ? rows[row] : -1;
            val[i] = lds128(src + row * kOutRow);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (at[i] >= 0)
              *reinterpret_cast<uint4*>(dst + static_cast<size_t>(at[i]) * a.out_ld) = val[i];
        }
      }
      rows = rows == s_row ? s_row + kTcRows : s_row;
    }
  } else if (warp >= kTcLoadWarp && warp < kTcCopyWarp) {
    // A slot is up to 32 copies of four rows, dealt out to these warps.  A unit's row
    // numbers are uniform values of the warp and one elected lane issues its copies:
    // issued from eight lanes they took 80 cycles each.  Columns past the last record
    // get the first record's row: no output is taken from them.
    constexpr int kShare = 32 / kTcLoadWarps;
    const int me = warp - kTcLoadWarp;
    const uint32_t leader = elect_one();
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int w = blockIdx.x; ok && w < total; w += gridDim.x) {
      const TcUnit u = tc_unit(a, w, groups);
      if (!u.ok) continue;
      const int n = u.t.z - u.t.y, quads = ((n + 15) & ~15) / 4;
      // lane j has the rows of this warp's copy j
      const int mine = lane % kShare * kTcLoadWarps + me, k = mine / quads;
      const int r0 = 4 * (mine - k * quads);
      int row[4], rows[kShare][4], block[kShare];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int p = u.t.y + (r0 + j < n ? r0 + j : 0);
        row[j] = a.index != nullptr ? a.index[p] / a.index_div : p;
        if (row[j] < 0 || row[j] >= a.act_rows) {
          record_status(a.status, kErrBadRow);
          row[j] = 0;
        }
      }
#pragma unroll
      for (int c = 0; c < kShare; ++c) {
        block[c] = __shfl_sync(0xffffffffu, k, c);
#pragma unroll
        for (int j = 0; j < 4; ++j) rows[c][j] = __shfl_sync(0xffffffffu, row[j], c);
      }
      const int per = tc_blocks(n);
      for (int kb = 0; kb < nb; kb += per) {
        ok = mbar_wait_idle(&bempty[s], ph ^ 1u, abort_flag, a.status, kErrTimeoutEmpty);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int blocks = min(per, nb - kb);
        if (leader) {
          // copies me, me + 4, ... of the blocks * quads of this slot
          const int copies = (blocks * quads - me + kTcLoadWarps - 1) / kTcLoadWarps;
          mbar_arrive_expect_tx(&bfull[s], copies * 512);
          const uint32_t dst = smem_u32(sB) + s * kTcBBytes + me * 512;
#pragma unroll
          for (int c = 0; c < kShare; ++c) {
            if (block[c] < blocks)
              tma_gather4(dst + c * (kTcLoadWarps * 512), &tm_rows, &bfull[s],
                          (kb + block[c]) * 64, rows[c][0], rows[c][1], rows[c][2], rows[c][3]);
          }
        }
        __syncwarp();
        if (++s == kSlots) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
    if (*abort_flag && lane == 0) {
      // Let every copy still in flight land before the CTA exits: the slots before s
      // are in their current round, the others in the one before.
      for (uint32_t i = 0; i < kSlots; ++i) {
        if (i >= s && ph == 0) break;  // never filled
        const unsigned long long t0 = globaltimer_ns();
        while (!mbar_try_wait(&bfull[i], i < s ? ph : ph ^ 1u)) {
          if (globaltimer_ns() - t0 > kWaitLimitNs) break;
        }
      }
    }
  } else if (warp == kTcCopyWarp) {
    if (lane == 0) {
      // ---------------------------------------------- codes and group records
      // One tiled copy of sixteen packed tiles' codes and one of their records per
      // stage; past the matrix they bring the next expert's rows or zeros, which
      // no operand row uses.
      uint32_t rings = 0;
      bool ok = true;
      for (int w = blockIdx.x; ok && w < total; w += gridDim.x) {
        const TcUnit u = tc_unit(a, w, groups);
        if (!u.ok) continue;
        const int row = u.t.x * a.m.tiles + u.m * kTcTiles;
        for (int kb = 0; kb < nb; kb += kTcBlocks, ++rings) {
          const uint32_t rs = rings % kTcRing;
          if (!mbar_wait_idle(&qempty[rs], ((rings / kTcRing) & 1u) ^ 1u, abort_flag, a.status,
                              kErrTimeoutEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&qfull[rs], args.ring_bytes);
          uint8_t* dst = sRing + rs * args.ring_bytes;
          tma_load_2d(dst, &tm_codes, &qfull[rs], kb * (kW4BlockBytes / 8), row);
          tma_load_2d(dst + kTcCodeBytes, &tm_records, &qfull[rs],
                      ((2 * kb) >> a.m.gshift) * (8 * kRec / 4), row);
        }
      }
      if (*abort_flag) {
        // Let every copy still in flight land before the CTA exits.
        for (uint32_t i = rings > kTcRing ? rings - kTcRing : 0u; i < rings; ++i) {
          const unsigned long long t0 = globaltimer_ns();
          while (!mbar_try_wait(&qfull[i % kTcRing], (i / kTcRing) & 1u)) {
            if (globaltimer_ns() - t0 > kWaitLimitNs) break;
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------ MMA issuer
    // Each of the two warps issues the products of one operand, into an accumulator of
    // its own: with one warp for both, the 16 products of two blocks took 375 of 1250
    // cycles.  The whole warp walks the stages, so that addresses and descriptors are
    // uniform values, and one elected lane issues.  This loop is what the block
    // rate hangs on, and among busy warps every instruction of it costs ten cycles:
    // with votes, tests ahead and 64-bit addresses it took 1150 cycles for two blocks.
    // After an abort the waits return at once and the unit is finished on what the
    // stages hold.
    TcAcc acc;
    const int op = warp - kTcMmaWarp;
    const uint32_t leader = elect_one();
    // descriptor of a K-major 128-byte-swizzled tile, without its start address
    constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
    uint32_t p = 0, phase = 0, bs = 0, bph = 0;
    const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), bfull0 = smem_u32(bfull),
                   bempty0 = smem_u32(bempty), acc_full0 = smem_u32(acc_full);
    const uint32_t sb = smem_u32(sB), at0 = tmem + kTcOperandCol + op * 32;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      tc_wait(bar, parity, abort_flag, a.status, kErrTimeoutFull);
    };
    auto next_slot = [&]() {
      if (++bs == kSlots) {
        bs = 0;
        bph ^= 1u;
      }
    };
    int issued = -1;  // half of the last unit
    TcUnit next{};
    if (static_cast<int>(blockIdx.x) < total) next = tc_unit(a, blockIdx.x, groups);
    for (int w = blockIdx.x; w < total; w += gridDim.x) {
      const TcUnit u = next;
      if (w + static_cast<int>(gridDim.x) < total) next = tc_unit(a, w + gridDim.x, groups);
      if (!u.ok) continue;
      const int n = __shfl_sync(0xffffffffu, u.t.z - u.t.y, 0);
      const int per = tc_blocks(n), cols = (n + 15) & ~15;
      acc.take(cols);
      bool ok = true;
      for (int b = acc.first; ok && b <= acc.last; ++b) {
        ok = mbar_wait(&acc_empty[b], (acc.used[b] & 1u) ^ 1u, abort_flag, a.status,
                       kErrTimeoutAccEmpty);
        ++acc.used[b];
      }
      if (!__all_sync(0xffffffffu, ok && *abort_flag == 0)) break;
      issued = acc.first;
      ++acc.filled[issued];
      const uint32_t idesc = idesc_f16_f32(128, static_cast<uint32_t>(cols));
      const bool rows = op == 0 || SWIGLU || u.m * kTcTiles + 8 < a.m.tiles;  // of this operand
      const uint32_t d = tmem + (op == 0 ? acc.d0 : acc.d1);
      const uint32_t acc_bar = acc_full0 + issued * 8;
      bool add = false;
      for (int left = nb; left > 0;) {
        // a slot: the blocks of several pairs, or with more than 64 records one block
        wait(bfull0 + bs * 8, bph);
        uint32_t lo = tc_desc(sb + bs * kTcBBytes);
        for (int here = min(per, left); here > 0; here -= kTcBlocks) {
          uint32_t bar = bempty0 + bs * 8, first_bar = 0, lo1 = lo + cols * 8;
          if (per == 1 && left > 1) {  // the second block's slot
            first_bar = bar;
            next_slot();
            bar = bempty0 + bs * 8;
            lo1 = tc_desc(sb + bs * kTcBBytes);
            wait(bfull0 + bs * 8, bph);
          }
          wait(full0 + p * 8, phase);
          __syncwarp();  // no lane may fall a phase behind
          tc_fence_after();
          const uint32_t at = at0 + p * (kTcBlocks * 64);
          if (leader) {
            if (rows) {
              tc_block(d, at, lo, kDescHi, idesc, add);
              if (first_bar != 0) tc_commit32(first_bar);
              if (left > 1) tc_block(d, at + 64, lo1, kDescHi, idesc, true);
              tc_commit32(empty0 + p * 8);
              if (here <= kTcBlocks) tc_commit32(bar);
              if (left <= kTcBlocks) tc_commit32(acc_bar);
            } else {  // nothing of this operand to wait for
              if (first_bar != 0) tc_arrive32(first_bar);
              tc_arrive32(empty0 + p * 8);
              if (here <= kTcBlocks) tc_arrive32(bar);
              if (left <= kTcBlocks) tc_arrive32(acc_bar);
            }
          }
          add = true;
          lo += 2 * cols * 8;
          left -= kTcBlocks;
          p ^= 1u;
          phase ^= p ^ 1u;
        }
        next_slot();
      }
    }
    // Tensor memory is released below: the last unit's products have to be done,
    // which the epilogue may not have waited for after an abort.
    if (issued >= 0) {
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(&acc_full[issued], (acc.filled[issued] & 1u) ^ 1u)) {
        if (globaltimer_ns() - t0 > kWaitLimitNs) break;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kTcMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Rows of activations as fp16 multiples of a power of two of the row, which puts its
// largest value into [2^14, 2^15), or is 2^-112 where that value is below 2^-98.  A bf16
// value down to 2^-31 of the largest stays exact; an fp32 one is rounded by 2^-12 at most
// down to 2^-28 of the largest, and by 2^-39 of the largest below.  A row with an infinity
// or a NaN keeps its values as they are.  dst may be src (fp32): a warp writes a chunk of
// 4 KB below what it has read.  A warp for a row; HBM bounds it (6000 x 2048 bf16 9 us,
// 49 MB).
template <bool F32>
__global__ void __launch_bounds__(256) w4_rows_f16(const uint8_t* src, long long src_pitch, int rows,
                                                   const int* count, int vec, uint8_t* dst,
                                                   long long dst_pitch, float* factor) {
  constexpr int kHold = 8;  // 16-byte vectors of a lane at once
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int total = count != nullptr ? max(0, min(rows, *count)) : rows;
  for (long long row = blockIdx.x * 8ll + (threadIdx.x >> 5); row < total; row += gridDim.x * 8ll) {
    const uint4* in = reinterpret_cast<const uint4*>(src + row * src_pitch);
    uint8_t* out = dst + row * dst_pitch;
    uint4 v[kHold];
    auto load = [&](int base) {
#pragma unroll
      for (int j = 0; j < kHold; ++j) {
        const int at = base + lane + 32 * j;
        v[j] = at < vec ? in[at] : make_uint4(0, 0, 0, 0);
      }
    };
    uint32_t top = 0;  // the largest magnitude's bits
    for (int base = 0; base < vec; base += 32 * kHold) {
      load(base);
#pragma unroll
      for (int j = 0; j < kHold; ++j) {
        const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = F32 ? max(top, w[i] & 0x7fffffffu) : __vmaxu2(top, w[i] & 0x7fff7fffu);
      }
    }
    if (!F32) top = max(top & 0xffffu, top >> 16) << 16;
    top = __reduce_max_sync(0xffffffffu, top);
    const int e = static_cast<int>(top >> 23);  // biased exponent
    const int shift = e == 255 ? 0 : min(141 - e, 112);
    const float mul = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
    if (lane == 0) factor[row] = __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
    for (int base = 0; base < vec; base += 32 * kHold) {
      if (vec > 32 * kHold) load(base);
      __syncwarp();  // the whole chunk is read
#pragma unroll
      for (int j = 0; j < kHold; ++j) {
        const int at = base + lane + 32 * j;
        const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
        if (F32) {
          if (at < vec)
            *reinterpret_cast<uint2*>(out + at * 8) =
                make_uint2(pack_f16x2(__uint_as_float(w[0]) * mul, __uint_as_float(w[1]) * mul),
                           pack_f16x2(__uint_as_float(w[2]) * mul, __uint_as_float(w[3]) * mul));
        } else if (at < vec) {
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[i] = pack_f16x2(__uint_as_float(w[i] << 16) * mul,
                              __uint_as_float(w[i] & 0xffff0000u) * mul);
          *reinterpret_cast<uint4*>(out + at * 16) = make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
      __syncwarp();
    }
  }
}

template <bool F32>
int rows_f16(const void* src, int rows, const int* count, int columns, void* dst,
             long long dst_pitch, float* factor, cudaStream_t stream) {
  const int vec = columns / (F32 ? 4 : 8);
  const int grid = std::min(rows / 8 + 1, 8 * device_sm_count());
  return note_cuda_error(launch_pdl(w4_rows_f16<F32>, dim3(grid), dim3(256), 0, stream,
                                    static_cast<const uint8_t*>(src),
                                    static_cast<long long>(columns) * (F32 ? 4 : 2), rows, count, vec,
                                    static_cast<uint8_t*>(dst), dst_pitch, factor)) == cudaSuccess
             ? kRcOk
             : kRcCudaError;
}

template <bool SWIGLU, bool HALVES, bool ZEROS>
int tc_launch(const W4Args& a, long long pitch, cudaStream_t stream) {
  TcArgs t{};
  t.a = a;
  t.rec_stride = (4 >> a.m.gshift) * 8 * a.m.rec;
  t.ring_bytes = kTcCodeBytes + kTcTiles * t.rec_stride;
  const int sh =
      1024 + kTcSlots<SWIGLU> * kTcBBytes + kTcRows * kTcOutRow<SWIGLU> + kTcRing * t.ring_bytes + 512 + kTcRows * 12;
  constexpr int kMost = 1024 + kTcSlots<SWIGLU> * kTcBBytes + kTcRows * kTcOutRow<SWIGLU> +
                        kTcRing * (kTcCodeBytes + kTcTiles * 256) + 512 + kTcRows * 12;
  static_assert(kMost <= 227 * 1024, "shared memory");
  static std::atomic<uint64_t> attr{0};
  if (!allow_smem(w4_tc<SWIGLU, HALVES, ZEROS>, kMost, attr)) return kRcCudaError;
  // x of a copy is a multiple of 16 bytes: blocks of 512, records of 8 rows of 4 or 8
  CUtensorMap codes, records, act;
  const long long rows = static_cast<long long>(a.E) * a.m.tiles;
  int rc = map_rows(&codes, a.m.q, 8, a.m.nb * (kW4BlockBytes / 8), rows,
                    kTcBlocks * kW4BlockBytes / 8, kTcTiles);
  if (rc == kRcOk)
    rc = map_rows(&records, a.m.s, 4, a.m.ng * 8 * a.m.rec / 4, rows, t.rec_stride / 4, kTcTiles);
  if (rc == kRcOk) rc = map_gather_rows(&act, a.act, a.act_rows, a.m.nb * 64, pitch);
  if (rc != kRcOk) return rc;
  const long long units =
      static_cast<long long>(a.max_tiles) * ((a.m.tiles + kTcTiles - 1) / kTcTiles);
  const int grid = static_cast<int>(std::min<long long>(units, device_sm_count()));
  return note_cuda_error(launch_pdl(w4_tc<SWIGLU, HALVES, ZEROS>, dim3(grid), dim3(kTcThreads), sh,
                                    stream, codes, records, act, t)) == cudaSuccess
             ? kRcOk
             : kRcCudaError;
}

template <bool SWIGLU>
int tc_dispatch(const W4Args& a, long long pitch, cudaStream_t stream) {
  if (a.m.gshift == 0)
    return a.m.rec == 8 ? tc_launch<SWIGLU, true, true>(a, pitch, stream)
                        : tc_launch<SWIGLU, true, false>(a, pitch, stream);
  return a.m.rec == 8 ? tc_launch<SWIGLU, false, true>(a, pitch, stream)
                      : tc_launch<SWIGLU, false, false>(a, pitch, stream);
}

}  // namespace

int w4_gemm(W4Args a, bool swiglu, const W4Rows& rows, bool f32, cudaStream_t stream) {
  const int columns = 64 * a.m.nb;
  // fp32 rows turn into fp16 ones in the first half of their place
  void* f16 = f32 ? const_cast<uint32_t*>(a.act) : rows.f16;
  const long long pitch = static_cast<long long>(columns) * (f32 ? 4 : 2);
  const int rc = f32 ? rows_f16<true>(a.act, a.act_rows, rows.count, columns, f16, pitch,
                                      rows.factor, stream)
                     : rows_f16<false>(a.act, a.act_rows, rows.count, columns, f16, pitch,
                                       rows.factor, stream);
  if (rc != kRcOk) return rc;
  a.act = static_cast<const uint32_t*>(f16);
  a.act_factor = rows.factor;
  return swiglu ? tc_dispatch<true>(a, pitch, stream) : tc_dispatch<false>(a, pitch, stream);
}

}  // namespace moe
