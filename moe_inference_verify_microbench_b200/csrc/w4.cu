// Grouped products with 4-bit expert weights (layout: w4.cuh).
//
//   w4_stream<true>   h[p] = silu(A[p] . Wg[e]) * (A[p] . Wu[e]), A[p] =
//                     src[index[p] / index_div]
//   w4_stream<false>  out[row_map[p]] = row_scale[row_map[p]] * (h[p] . Wd[e])
//
// At few records per expert these are a stream of weights: 0.5 byte and the
// group's share of a scale per weight, so HBM bounds them and everything else
// has to stay below 23 bytes of weights per cycle and SM.  One persistent CTA of
// sixteen warps per SM.  Every warp copies the part of a 16-row tile that it will
// use itself (contiguous, in the order its lanes consume) into shared memory
// with cp.async, several tiles ahead, so the stream needs no barrier; it turns
// codes into fp16 operands in registers (20 integer instructions per 1024
// weights, no conversion) and multiplies them on the tensor cores as the 16-row
// operand of mma.m16n8k16, with up to 16 records as its columns.  The records'
// rows stay in registers for all tiles of an expert.  The warps that share a
// tile along K add their fp32 partials through shared memory.
//
// Numerics: products of activations with (q - z) are exact in fp32; each
// group (or a warp's share of it) is summed on the tensor cores in fp32 and
// then scaled in fp32, so no weight is ever rounded to bf16.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "grouped_gemm.cuh"
#include "internal.h"
#include "w4.cuh"

namespace moe {

// ------------------------------------------------------------------ packing

struct W4PackArgs {
  const uint8_t* codes[2];  // [E][N][K]; [1] null: one matrix in 16-row tiles
  const uint16_t* scales[2];
  const uint8_t* zeros[2];
  int E, N, K, group;
  uint8_t* q;
  uint16_t* s;
  int* status;
};

// The word of a lane's eight columns 8i + {0, 1} from `codes`.
__device__ __forceinline__ uint32_t w4_word(const uint8_t* codes, bool& bad) {
  uint32_t w = 0, seen = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = *reinterpret_cast<const uint16_t*>(codes + 8 * i);
    seen |= v;
    w |= (v & 0xfu) << (4 * i) | ((v >> 8) & 0xfu) << (4 * i + 16);
  }
  bad |= (seen & 0xf0f0u) != 0;
  return w;
}

__global__ void __launch_bounds__(256) w4_pack(const W4PackArgs a) {
  pdl_wait();
  pdl_trigger();
  const int nb = a.K / 64, ng = a.K / a.group;
  const bool pair = a.codes[1] != nullptr;
  const int rows = pair ? 8 : 16;  // rows of each matrix per tile
  const int tiles = a.N / rows;
  const long long words = static_cast<long long>(a.E) * tiles * nb * 32;
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  const long long i0 = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  bool bad = false;
  for (long long i = i0; i < words; i += step) {
    const int lane = static_cast<int>(i & 31);
    const long long blk = i >> 5;
    const int kb = static_cast<int>(blk % nb);
    const long long et = blk / nb;  // expert * tiles + tile
    const int tile = static_cast<int>(et % tiles);
    const long long e = et / tiles;
    const int g = lane >> 2, t = lane & 3;
    const size_t row = static_cast<size_t>(e) * a.N + static_cast<size_t>(tile) * rows + g;
    const size_t col = static_cast<size_t>(kb) * 64 + 2 * t;
    const uint8_t* p0 = a.codes[0] + row * a.K + col;
    const uint8_t* p1 = pair ? a.codes[1] + row * a.K + col : p0 + static_cast<size_t>(8) * a.K;
    uint4 w;
    w.x = w4_word(p0, bad);
    w.y = w4_word(p0 + 32, bad);
    w.z = w4_word(p1, bad);
    w.w = w4_word(p1 + 32, bad);
    reinterpret_cast<uint4*>(a.q)[i] = w;
  }
  const long long sc = static_cast<long long>(a.E) * tiles * ng * 8;
  for (long long i = i0; i < sc; i += step) {
    const int g = static_cast<int>(i & 7);
    const long long b = i >> 3;
    const int grp = static_cast<int>(b % ng);
    const long long et = b / ng;
    const int tile = static_cast<int>(et % tiles);
    const long long e = et / tiles;
    const size_t row = static_cast<size_t>(e) * a.N + static_cast<size_t>(tile) * rows + g;
    const size_t o0 = row * ng + grp;
    const size_t o1 = pair ? o0 : o0 + static_cast<size_t>(8) * ng;
    const bool zp = a.zeros[0] != nullptr;
    uint16_t* rec = a.s + (zp ? 4 : 2) * i;
    rec[0] = a.scales[0][o0];
    rec[1] = a.scales[pair ? 1 : 0][o1];
    if (zp) {
      const uint8_t z0 = a.zeros[0][o0], z1 = a.zeros[pair ? 1 : 0][o1];
      bad |= z0 > 15 || z1 > 15;
      rec[2] = 0x6400u | (z0 & 15u);  // fp16 1024 + z
      rec[3] = 0x6400u | (z1 & 15u);
    }
  }
  if (bad) record_status(a.status, kErrBadCode);
}

// ------------------------------------------------------------------ streaming

// Work of a tile-table entry: its records in chunks of 8 NT, each chunk one pass
// over the expert's tiles (units).  A bad entry has none and is reported.
template <int NT>
__device__ __forceinline__ int w4_chunks(const W4Args& a, const int4& t) {
  if (!w4_entry_ok(a, t)) return 0;
  return static_cast<int>(static_cast<unsigned>(t.z - t.y + 8 * NT - 1) / (8u * NT));
}

// Cost of a unit: the stream of its weights, and a share for every eight
// records multiplied with them.
template <int NT>
__device__ __forceinline__ int w4_unit_cost(const int4& t) {
  return NT > 1 && t.z - t.y > 8 ? 5 : 4;
}

// A position in the work: tile-table entry, unit within it.
struct W4Pos {
  int entry, unit;
};

// This CTA's contiguous range of units [lo, hi), the summed cost split evenly
// over the grid.  Every thread of the CTA calls it.
template <int NT>
__device__ __forceinline__ void w4_range(const W4Args& a, int nt, W4Pos* lo, W4Pos* hi) {
  __shared__ long long sums[kW4Warps];
  __shared__ W4Pos pos[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto cost = [&](int i, int* per) -> long long {
    *per = 1;
    if (i >= nt) return 0;
    const int4 t = a.tiles[i];
    *per = w4_unit_cost<NT>(t);
    return static_cast<long long>(w4_chunks<NT>(a, t)) * (a.m.tiles * *per);
  };
  int per0;
  const long long first = cost(threadIdx.x, &per0);  // most tables fit the CTA
  long long mine = first;
  for (int i = threadIdx.x + kW4Threads; i < nt; i += kW4Threads) {
    int per;
    mine += cost(i, &per);
  }
  if (threadIdx.x < 2) pos[threadIdx.x] = {0, 0};
  long long total = 0, carry = 0;
  for (int base = 0; base < nt; base += kW4Threads) {
    int per = per0;
    const long long c = base == 0 ? first : cost(base + static_cast<int>(threadIdx.x), &per);
    long long incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (base == 0) {  // the grand total, once
      long long all = nt <= kW4Threads ? incl : mine;
      if (nt > kW4Threads) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      }
      if (lane == 31) sums[warp] = all;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int w = 0; w < kW4Warps; ++w) total += sums[w];
    }
    if (nt > kW4Threads) {
      __syncthreads();
      if (lane == 31) sums[warp] = incl;
      __syncthreads();
    }
    long long before = carry;
#pragma unroll
    for (int w = 0; w < kW4Warps; ++w) {
      if (w < warp) before += sums[w];
      carry += sums[w];
    }
    incl += before;
    const long long excl = incl - c;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long long want = total * (static_cast<long long>(blockIdx.x) + k) / gridDim.x;
      if (want > excl && want <= incl)
        pos[k] = {base + static_cast<int>(threadIdx.x),
                  static_cast<int>((want - excl + per - 1) / per)};
    }
  }
  __syncthreads();
  *lo = pos[0];
  *hi = pos[1];
}

// Walks the units of a range, every tl-th from a first one on, in runs of tiles
// that share their expert and records.
template <int NT>
struct W4Walk {
  int entry, chunk, tile;  // next unit
  int chunks;              // of the entry
  int4 t;
  __device__ __forceinline__ void open(const W4Args& a, int nt) {
    for (chunks = 0; entry < nt; ++entry) {
      t = a.tiles[entry];
      chunks = w4_chunks<NT>(a, t);
      if (chunks > 0) return;
    }
  }
  __device__ __forceinline__ void start(const W4Args& a, int nt, const W4Pos& lo, int skip) {
    entry = lo.entry;
    chunk = 0;
    tile = lo.unit + skip;
    open(a, nt);
  }
  // Tiles of the run that starts at the next unit: 0 at the end of the range.
  __device__ __forceinline__ int run(const W4Args& a, int nt, const W4Pos& hi) {
    while (tile >= a.m.tiles && entry < nt) {
      tile -= a.m.tiles;
      if (++chunk >= chunks) {
        chunk = 0;
        ++entry;
        open(a, nt);
      }
    }
    if (entry >= nt || entry > hi.entry) return 0;
    const int end =
        entry == hi.entry ? min(a.m.tiles, hi.unit - chunk * a.m.tiles) : a.m.tiles;
    return end > tile ? (end - tile + a.p.tl - 1) >> a.p.tl_shift : 0;
  }
};

template <int BYTES>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES)
               : "memory");
}

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// d += (codes of a half block's two words) . records, two of the block's four
// 16-column steps.  Without FOLD the zero points come off the operands first:
// z holds 1024 + z of rows g and g + 8 in the halves.
template <int NT, bool FOLD>
__device__ __forceinline__ void w4_half(float (&d)[NT][4], uint32_t wl, uint32_t wh, int h,
                                        const uint32_t (&b)[NT][8], uint32_t z) {
  uint32_t lo[4], hi[4];
  w4_pairs(wl, lo);
  w4_pairs(wh, hi);
  if constexpr (!FOLD) {
    const uint32_t zl = __byte_perm(z, 0, 0x1010), zh = __byte_perm(z, 0, 0x3232);
    const uint32_t yl = (zl & 0x000f000fu) << 4 | 0x54005400u;  // 64 + z
    const uint32_t yh = (zh & 0x000f000fu) << 4 | 0x54005400u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = sub_f16x2(lo[i], (i & 1) ? yl : zl);
      hi[i] = sub_f16x2(hi[i], (i & 1) ? yh : zh);
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int j = 0; j < NT; ++j)
      mma_16816(d[j], lo[2 * s], hi[2 * s], lo[2 * s + 1], hi[2 * s + 1], b[j][4 * h + 2 * s],
                b[j][4 * h + 2 * s + 1]);
}

// acc += scale * d: the end of a group (or of the warp's share of it).
template <int NT>
__device__ __forceinline__ void w4_flush(float (&acc)[NT][4], const float (&d)[NT][4],
                                         uint32_t sc) {
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc[j][c] = fmaf(c < 2 ? bf16_lo(sc) : bf16_hi(sc), d[j][c], acc[j][c]);
}

// What of a tile is this warp's.
struct W4Share {
  int ks, tl;    // its place along K, its place among the tiles worked on at once
  int kb0, myb;  // its blocks
  int g0;        // the first group they touch
};

template <int KB>
__device__ __forceinline__ W4Share w4_share(const W4Args& a) {
  // the shuffle tells the compiler that these are the same for the whole warp
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  W4Share s;
  s.ks = warp & (a.p.ks - 1);
  s.tl = warp >> a.p.ks_shift;
  s.myb = max(0, min(KB, a.m.nb - s.ks * KB));
  s.kb0 = s.myb > 0 ? s.ks * KB : 0;  // a warp without blocks multiplies with zeros
  s.g0 = (2 * s.kb0) >> a.m.gshift;
  return s;
}

// A chunk's activations as this warp's matrix operand in fp16: its blocks of
// records rec0 .. rec0 + n (zeros past n and past the last block).  A record's
// part is scaled by the power of two that puts its largest magnitude in [2^15,
// 2^16), and `inv` takes it back: a bf16 value within 2^-32 of the largest keeps
// all its bits, a smaller one loses at most 2^-40 of the largest.
//
// Without zero points the weight operand stays 1024 + q or 64 + q, and a group's
// sum starts at -(1032 or 72) times its activations (`fold`), so the subtraction
// costs nothing per weight; it cancels to within 2^-23 * 1032 * sum|x|.
// kW4Half subtracts from every operand instead, which is exact.
template <int KB, int NT, int MODE>
__device__ __forceinline__ void w4_load_records(const W4Args& a, const W4Share& sh, int rec0,
                                                int n, uint32_t (&b)[KB][NT][8],
                                                float (&fold)[KB][NT][2], float (&inv)[NT][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    int row = -1;
    const int rec = 8 * j + g;
    if (rec < n) {
      row = a.index != nullptr ? a.index[rec0 + rec] / a.index_div : rec0 + rec;
      if (row < 0 || row >= a.act_rows) {
        record_status(a.status, kErrBadRow);
        row = -1;
      }
    }
    const uint32_t* src = a.act + (static_cast<size_t>(max(row, 0)) * a.m.nb + sh.kb0) * 32 + t;
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const bool have = row >= 0 && k < sh.myb;
#pragma unroll
      for (int i = 0; i < 8; ++i) b[k][j][i] = have ? __ldg(src + k * 32 + 4 * i) : 0u;
    }
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) most = __vmaxu2(most, b[k][j][i] & 0x7fff7fffu);
    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = static_cast<int>(max(most & 0xffffu, most >> 16) >> 7);  // biased exponent
    const int up = min(142 - e, 110);
    const float scale = __int_as_float((127 + up) << 23);
    const float back = __int_as_float((127 - up) << 23);
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t v = b[k][j][i];
        const __half2 h = __floats2half2_rn(bf16_lo(v) * scale, bf16_hi(v) * scale);
        b[k][j][i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    // of this lane's columns: records 8j + 2t and 8j + 2t + 1
    inv[j][0] = __shfl_sync(0xffffffffu, back, 8 * t);
    inv[j][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
  }
  if constexpr (MODE != kW4Half) {
    // a product with the operand of codes 8, per group: kept at its first block
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = KB - 1; k >= 0; --k) {
        if (MODE == kW4Block || (k & 1)) d[0] = d[1] = d[2] = d[3] = 0.0f;
#pragma unroll
        for (int st = 0; st < 4; ++st)
          mma_16816(d, 0x64086408u, 0x64086408u, 0x54805480u, 0x54805480u, b[k][j][2 * st],
                    b[k][j][2 * st + 1]);
        fold[k][j][0] = -d[0];
        fold[k][j][1] = -d[1];
      }
    }
  }
}

// acc = this warp's share of a tile (its codes at `slot`, its group records at
// slot + KB blocks) times the records.
template <int KB, int NT, int MODE>
__device__ __forceinline__ void w4_tile(const W4Args& a, const W4Share& sh, uint32_t slot,
                                        const uint32_t (&b)[KB][NT][8],
                                        const float (&fold)[KB][NT][2],
                                        const float (&inv)[NT][2], float (&acc)[NT][4]) {
  const int lane = threadIdx.x & 31;
  const uint32_t qp = slot + lane * 16;
  const uint32_t rec = slot + KB * kW4BlockBytes + (lane >> 2) * a.m.rec;
  const uint32_t step = 8 * a.m.rec;
  float d[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
#pragma unroll
  for (int k = 0; k < KB; ++k) {
    const uint4 w = lds128(qp + k * kW4BlockBytes);
    if (MODE != kW4TwoBlocks || (k & 1) == 0) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) d[j][c] = MODE != kW4Half ? fold[k][j][c & 1] : 0.0f;
    }
    if constexpr (MODE != kW4Half) {
      w4_half<NT, true>(d, w.x, w.z, 0, b[k], 0u);
      w4_half<NT, true>(d, w.y, w.w, 1, b[k], 0u);
      if (MODE == kW4TwoBlocks && (k & 1)) w4_flush<NT>(acc, d, lds32(rec + (k >> 1) * step));
      // a group of 128 may span two of an odd number of blocks: its record serves both
      if (MODE == kW4Block)
        w4_flush<NT>(acc, d, lds32(rec + (((2 * (sh.kb0 + k)) >> a.m.gshift) - sh.g0) * step));
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t r = rec + (((2 * (sh.kb0 + k) + h) >> a.m.gshift) - sh.g0) * step;
        const uint32_t z = a.m.rec == 8 ? lds32(r + 4) : 0x64086408u;
        w4_half<NT, false>(d, h == 0 ? w.x : w.y, h == 0 ? w.z : w.w, h, b[k], z);
        w4_flush<NT>(acc, d, lds32(r));
        if (h == 0) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) d[j][c] = 0.0f;
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[j][c] *= inv[j][c & 1];
}

// The groups that KB blocks touch at most.
constexpr int w4_groups(int kb, int gshift) { return ((2 * kb - 2) >> gshift) + 2; }

// Copies this warp's share of a tile into a slot (asynchronously): codes from q
// on, group records from s on.  Blocks past the last are left as they are (any
// code times zero is zero), but every record that is read is a real one.
template <int KB>
__device__ __forceinline__ void w4_fetch(const W4Args& a, const W4Share& sh, uint32_t slot,
                                         const uint8_t* q, const uint8_t* s) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < KB; ++k)
    if (k < sh.myb) cp_async_16(slot + lane * 16 + k * kW4BlockBytes, q + k * kW4BlockBytes, 16);
  const uint32_t dst = slot + KB * kW4BlockBytes + lane * a.m.rec;
  const int groups = w4_groups(KB, a.m.gshift);
  for (int i = lane >> 3; i < groups; i += 4) {  // four groups of eight records at a time
    const int from = min(i, a.m.ng - 1 - sh.g0) - (lane >> 3), o = (i - (lane >> 3)) * 8 * a.m.rec;
    if (a.m.rec == 8) cp_async_small<8>(dst + o, s + from * 64);
    else cp_async_small<4>(dst + o, s + from * 32);
  }
}

// The units [lo, hi) of the tile table on this CTA, NT * 8 records to a chunk at
// most.  Each group of ks warps takes every tl-th unit.
template <bool SWIGLU, int KB, int NT, int SLOTS, int MODE>
__device__ __forceinline__ void w4_units(const W4Args& a, uint8_t* smem, float* part, int nt,
                                         const W4Pos& lo, const W4Pos& hi) {
  const W4Plan& p = a.p;
  const W4Share sh = w4_share<KB>(a);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warp = sh.tl * p.ks + sh.ks;
  const uint32_t base = smem_u32(smem) + warp * SLOTS * p.slot_bytes;
  W4Walk<NT> f, c;  // the next run to fetch, the run to work on
  c.start(a, nt, lo, sh.tl);
  f = c;
  const uint8_t* fq = nullptr;  // next tile to fetch
  const uint8_t* fsrc = nullptr;
  int left = f.run(a, nt, hi);
  uint32_t fslot = base, slot = base;
  const uint32_t end_slot = base + SLOTS * p.slot_bytes;
  const int q_tile = a.m.nb * kW4BlockBytes, s_tile = a.m.ng * 8 * a.m.rec;
  auto aim = [&]() {  // pointers of the run's first tile
    const size_t et = static_cast<size_t>(f.t.x) * a.m.tiles + f.tile;
    fq = a.m.q + et * q_tile + sh.kb0 * kW4BlockBytes + lane * 16;
    fsrc = a.m.s + et * s_tile + (sh.g0 * 8 + lane) * a.m.rec;
  };
  if (left > 0) aim();
  auto fetch = [&]() {
    if (left > 0) {
      w4_fetch<KB>(a, sh, fslot, fq, fsrc);
      fq += static_cast<size_t>(q_tile) << p.tl_shift;
      fsrc += static_cast<size_t>(s_tile) << p.tl_shift;
      f.tile += p.tl;
      if (--left == 0) {
        left = f.run(a, nt, hi);
        if (left > 0) aim();
      }
    }
    cp_async_commit();
    fslot += p.slot_bytes;
    if (fslot == end_slot) fslot = base;
  };
#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i) fetch();
  constexpr int kStride = NT * 128;
  constexpr int kBuffer = kW4Warps * kStride;
  int buffer = 0;
  for (int count; (count = c.run(a, nt, hi)) > 0;) {
    const int rec0 = c.t.y + c.chunk * (8 * NT), n = min(8 * NT, c.t.z - rec0);
    auto pass = [&](auto nt_c) {
      constexpr int N = decltype(nt_c)::value;
      uint32_t b[KB][N][8];
      float fold[KB][N][2], inv[N][2];
      w4_load_records<KB, N, MODE>(a, sh, rec0, n, b, fold, inv);
      // Value pairs u = 2j + c (records 8j + 2t + c) are stored by the warps u
      // modulo ks: their rows (-1: none) and scales.
      int orow[2 * N];
      float scale[2 * N];
#pragma unroll
      for (int u = 0; u < 2 * N; ++u) {
        const int rec = 8 * (u >> 1) + 2 * t + (u & 1);
        orow[u] = -1;
        scale[u] = 1.0f;
        if ((u & (p.ks - 1)) == sh.ks && rec < n) {
          orow[u] = rec0 + rec;
          if (!SWIGLU && a.row_map != nullptr) orow[u] = __ldg(a.row_map + rec0 + rec);
          if (orow[u] < 0 || orow[u] >= a.out_rows) {
            record_status(a.status, kErrBadRow);
            orow[u] = -1;
          } else if (!SWIGLU && a.row_scale != nullptr) {
            scale[u] = __ldg(a.row_scale + orow[u]);
          }
        }
      }
      __nv_bfloat16* out = a.out + c.tile * (SWIGLU ? 8 : 16) + g;
      for (int i = 0; i < count; ++i) {
        cp_async_wait_group<SLOTS - 2>();
        __syncwarp();  // every lane's copies have landed, and the last tile's slot is free
        fetch();
        float acc[N][4];
        w4_tile<KB, N, MODE>(a, sh, slot, b, fold, inv, acc);
        slot += p.slot_bytes;
        if (slot == end_slot) slot = base;
        if (p.ks > 1) {
          // The ks partials of the tile meet in shared memory: [buffer][warp][value]
          // [lane], two buffers so that one barrier per tile suffices.
          float* pw = part + buffer + warp * kStride + lane;
#pragma unroll
          for (int j = 0; j < N; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) pw[(4 * j + v) * 32] = acc[j][v];
          named_barrier(1 + sh.tl, p.ks * 32);
        }
#pragma unroll
        for (int u = 0; u < 2 * N; ++u) {
          if ((u & (p.ks - 1)) == sh.ks) {
            float v0 = acc[u >> 1][u & 1], v1 = acc[u >> 1][(u & 1) + 2];
            if (p.ks > 1) {
              v0 = v1 = 0.0f;
              const float* pr =
                  part + buffer + sh.tl * p.ks * kStride + (4 * (u >> 1) + (u & 1)) * 32 + lane;
              for (int w = 0; w < p.ks; w += 2) {
                v0 += pr[0] + pr[kStride];
                v1 += pr[64] + pr[kStride + 64];
                pr += 2 * kStride;
              }
            }
            if (orow[u] >= 0) {
              __nv_bfloat16* dst = out + static_cast<size_t>(orow[u]) * a.out_ld;
              if constexpr (SWIGLU) {
                dst[0] = __float2bfloat16_rn(silu_f(v0) * v1);
              } else {
                dst[0] = __float2bfloat16_rn(v0 * scale[u]);
                dst[8] = __float2bfloat16_rn(v1 * scale[u]);
              }
            }
          }
        }
        out += p.tl * (SWIGLU ? 8 : 16);
        buffer ^= kBuffer;
      }
    };
    if (NT > 1 && n > 8) pass(std::integral_constant<int, NT>{});
    else pass(std::integral_constant<int, 1>{});
    c.tile += count * p.tl;
  }
  cp_async_wait_all();  // nothing is in flight when the CTA exits
}

template <int NT>
constexpr int w4_part_bytes() {
  return 2 * kW4Warps * NT * 128 * 4;
}
constexpr int kW4SmemBytes = 224 * 1024;

template <bool SWIGLU, int KB, int NT, int SLOTS, int MODE>
__global__ void __launch_bounds__(kW4Threads, 1) w4_stream(const W4Args a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  pdl_wait();
  pdl_trigger();
  const int nt = max(0, min(*a.num_tiles, a.max_tiles));
  W4Pos lo, hi;
  w4_range<NT>(a, nt, &lo, &hi);
  if constexpr (!SWIGLU) w4_zero_tail(a, threadIdx.x, kW4Threads);
  w4_units<SWIGLU, KB, NT, SLOTS, MODE>(a, smem_raw + w4_part_bytes<NT>(),
                                         reinterpret_cast<float*>(smem_raw), nt, lo, hi);
}

// ------------------------------------------------------------------ launchers

// Cuts a projection over the warps, kb blocks to each.
static W4Plan w4_plan(const W4Matrix& m, int kb) {
  W4Plan p{};
  p.ks = 1;
  while (p.ks * kb < m.nb) p.ks *= 2;
  p.tl = kW4Warps / p.ks;
  while ((1 << p.ks_shift) < p.ks) ++p.ks_shift;
  while ((1 << p.tl_shift) < p.tl) ++p.tl_shift;
  p.slot_bytes = kb * kW4BlockBytes + w4_groups(kb, m.gshift) * 8 * m.rec;
  return p;
}

// Of the block counts the kernels are built for, the one that leaves the fewest
// slots idle (then the largest: fewer warps share a tile and add their partials).
static int w4_best_kb(int nb, std::initializer_list<int> kbs) {
  int best = 0, best_slots = 0;
  for (const int kb : kbs) {
    int ks = 1;
    while (ks * kb < nb) ks *= 2;
    if (ks <= kW4Warps && (best == 0 || ks * kb <= best_slots)) {
      best = kb;
      best_slots = ks * kb;
    }
  }
  return best;
}

static W4Matrix w4_matrix(const W4Bank& bank, bool down) {
  W4Matrix m{};
  m.q = static_cast<const uint8_t*>(down ? bank.w2_q : bank.w13_q);
  m.s = static_cast<const uint8_t*>(down ? bank.w2_s : bank.w13_s);
  m.rec = bank.zeros ? 8 : 4;
  m.tiles = down ? bank.H / 16 : bank.I / 8;
  const int K = down ? bank.I : bank.H;
  m.nb = K / 64;
  m.ng = K / bank.group;
  m.gshift = bank.group == 32 ? 0 : bank.group == 64 ? 1 : 2;
  return m;
}

int w4_check_bank(const W4Bank& b) {
  if (b.E <= 0 || b.H <= 0 || b.I <= 0 || b.w13_q == nullptr || b.w13_s == nullptr ||
      b.w2_q == nullptr || b.w2_s == nullptr)
    return kRcBadArgument;
  if (b.group != 32 && b.group != 64 && b.group != 128) return kRcUnsupported;
  if (b.H % 64 != 0 || b.I % 64 != 0 || b.H % b.group != 0 || b.I % b.group != 0 ||
      b.H > kW4MaxK || b.I > kW4MaxK || b.E > 1024)
    return kRcUnsupported;
  for (const void* p : {b.w13_q, b.w13_s, b.w2_q, b.w2_s})
    if (!aligned16(p)) return kRcBadArgument;
  return kRcOk;
}

template <bool SWIGLU, int KB, int NT, int SLOTS, int MODE>
static int w4_launch(W4Args& a, cudaStream_t stream) {
  a.p = w4_plan(a.m, KB);
  const int sh = w4_part_bytes<NT>() + kW4Warps * SLOTS * a.p.slot_bytes;
  if (sh > kW4SmemBytes) return kRcUnsupported;
  static std::atomic<uint64_t> attr{0};
  if (!allow_smem(w4_stream<SWIGLU, KB, NT, SLOTS, MODE>, kW4SmemBytes, attr)) return kRcCudaError;
  const long long units = static_cast<long long>(a.max_tiles) * a.m.tiles;
  const int grid = static_cast<int>(std::min<long long>(units, device_sm_count()));
  return note_cuda_error(launch_pdl(w4_stream<SWIGLU, KB, NT, SLOTS, MODE>, dim3(grid),
                                    dim3(kW4Threads), sh, stream, a)) == cudaSuccess
             ? kRcOk
             : kRcCudaError;
}

template <bool SWIGLU, int MODE>
static int w4_dispatch_mode(W4Args& a, cudaStream_t stream) {
  // Up to about six records per expert a pass takes eight, so that a warp can
  // hold twice the blocks and half as many warps add partials; beyond, sixteen.
  const int wide = a.avg > 6 ? w4_best_kb(a.m.nb, {2, 3, 4}) : 0;
  constexpr int kSlots8 = MODE == kW4Half ? 2 : 3;
  switch (wide) {
    case 2: return w4_launch<SWIGLU, 2, 2, 8, MODE>(a, stream);
    case 3: return w4_launch<SWIGLU, 3, 2, 5, MODE == kW4TwoBlocks ? kW4Block : MODE>(a, stream);
    case 4: return w4_launch<SWIGLU, 4, 2, 4, MODE>(a, stream);
  }
  switch (w4_best_kb(a.m.nb, {4, 6, 8})) {
    case 4: return w4_launch<SWIGLU, 4, 1, 4, MODE>(a, stream);
    case 6: return w4_launch<SWIGLU, 6, 1, 3, MODE>(a, stream);
    case 8: return w4_launch<SWIGLU, 8, 1, kSlots8, MODE>(a, stream);
  }
  return kRcUnsupported;
}

template <bool SWIGLU>
static int w4_dispatch(W4Args& a, cudaStream_t stream) {
  // Whole layers, 128 experts of 2048 x 768, group 128: at 4 records per expert the
  // stream takes 110 us and the tensor-memory form 140, at 8 they take 152 and 146.
  if (a.avg >= kW4TcRecords) return w4_gemm(a, SWIGLU, stream);
  if (a.m.rec == 8 || a.m.gshift == 0) return w4_dispatch_mode<SWIGLU, kW4Half>(a, stream);
  if (a.m.gshift == 1) return w4_dispatch_mode<SWIGLU, kW4Block>(a, stream);
  return w4_dispatch_mode<SWIGLU, kW4TwoBlocks>(a, stream);
}

int launch_w4_w13(const W4Bank& bank, const void* src, int src_rows, const int* index,
                  int index_div, int M, const int4* tiles, const int* num_tiles, int max_tiles,
                  void* h_out, int avg, int* status, cudaStream_t stream) {
  if (const int rc = w4_check_bank(bank); rc != kRcOk) return rc;
  if (M < 0 || max_tiles < 0 || index_div <= 0 || src_rows < 0 || tiles == nullptr ||
      num_tiles == nullptr)
    return kRcBadArgument;
  if (M == 0 || max_tiles == 0) return kRcOk;
  if (src == nullptr || h_out == nullptr || !aligned16(src) || !aligned16(h_out)) return kRcBadArgument;
  W4Args a{};
  a.m = w4_matrix(bank, false);
  a.act = static_cast<const uint32_t*>(src);
  a.act_rows = src_rows;
  a.index = index;
  a.index_div = index_div;
  a.M = M;
  a.tiles = tiles;
  a.num_tiles = num_tiles;
  a.max_tiles = max_tiles;
  a.E = bank.E;
  a.out = static_cast<__nv_bfloat16*>(h_out);
  a.out_ld = bank.I;
  a.out_rows = M;
  a.avg = avg;
  a.status = status;
  return w4_dispatch<true>(a, stream);
}

int launch_w4_w2(const W4Bank& bank, const void* h, int M, const int4* tiles, const int* num_tiles,
                 int max_tiles, const int* row_map, const float* row_scale, void* out,
                 int out_rows, int avg, int* status, cudaStream_t stream,
                 const long long* tail) {
  if (const int rc = w4_check_bank(bank); rc != kRcOk) return rc;
  if (M < 0 || max_tiles < 0 || out_rows < 0 || tiles == nullptr || num_tiles == nullptr)
    return kRcBadArgument;
  if (M == 0 || max_tiles == 0) return kRcOk;
  if (h == nullptr || out == nullptr || !aligned16(h) || !aligned16(out)) return kRcBadArgument;
  W4Args a{};
  a.m = w4_matrix(bank, true);
  a.act = static_cast<const uint32_t*>(h);
  a.act_rows = M;
  a.index_div = 1;
  a.M = M;
  a.tiles = tiles;
  a.num_tiles = num_tiles;
  a.max_tiles = max_tiles;
  a.E = bank.E;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.out_ld = bank.H;
  a.out_rows = out_rows;
  a.row_map = row_map;
  a.row_scale = row_scale;
  a.tail = tail;
  a.avg = avg;
  a.status = status;
  return w4_dispatch<false>(a, stream);
}

int launch_w4_pack(const uint8_t* codes0, const void* scales0, const uint8_t* zeros0,
                   const uint8_t* codes1, const void* scales1, const uint8_t* zeros1, int E, int N,
                   int K, int group, void* q, void* s, int* status, cudaStream_t stream) {
  if (codes0 == nullptr || scales0 == nullptr || q == nullptr || s == nullptr ||
      (codes1 == nullptr) != (scales1 == nullptr) ||
      (codes1 != nullptr && (zeros0 == nullptr) != (zeros1 == nullptr)) ||
      (codes1 == nullptr && zeros1 != nullptr) || E <= 0 || N <= 0 || K <= 0)
    return kRcBadArgument;
  if ((group != 32 && group != 64 && group != 128) || K % 64 != 0 || K % group != 0 ||
      K > kW4MaxK || N % (codes1 != nullptr ? 8 : 16) != 0 || E > 1024)
    return kRcUnsupported;
  if (!aligned16(q) || !aligned16(s) || !aligned16(codes0) || !aligned16(codes1))
    return kRcBadArgument;
  W4PackArgs a{};
  a.codes[0] = codes0;
  a.codes[1] = codes1;
  a.scales[0] = static_cast<const uint16_t*>(scales0);
  a.scales[1] = static_cast<const uint16_t*>(scales1);
  a.zeros[0] = zeros0;
  a.zeros[1] = zeros1;
  a.E = E;
  a.N = N;
  a.K = K;
  a.group = group;
  a.q = static_cast<uint8_t*>(q);
  a.s = static_cast<uint16_t*>(s);
  a.status = status;
  return note_cuda_error(launch_pdl(w4_pack, dim3(device_sm_count() * 8), dim3(256), 0, stream,
                                    a)) == cudaSuccess
             ? kRcOk
             : kRcCudaError;
}

}  // namespace moe
