// The streaming form of the grouped products with 4-bit weights: device code of the
// grouped kernels (w4.cu) and of the decode layer (w4_decode.cu).
#pragma once

#include <initializer_list>
#include <type_traits>

#include "grouped_gemm.cuh"
#include "w4.cuh"

namespace moe {

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

// A chunk's activations as this warp's matrix operand: from bf16 pairs (zeros past
// the last record and past the last block) to fp16 in place.  A record's part is
// scaled by the power of two that puts its largest magnitude in [2^15,
// 2^16), and `inv` takes it back: a bf16 value within 2^-32 of the largest keeps
// all its bits, a smaller one loses at most 2^-40 of the largest.
//
// Without zero points the weight operand stays 1024 + q or 64 + q, and a group's
// sum starts at -(1032 or 72) times its activations (`fold`), so the subtraction
// costs nothing per weight; it cancels to within 2^-23 * 1032 * sum|x|.
// kW4Half subtracts from every operand instead, which is exact.
template <int KB, int NT, int MODE>
__device__ __forceinline__ void w4_prepare_records(uint32_t (&b)[KB][NT][8],
                                                   float (&fold)[KB][NT][2],
                                                   float (&inv)[NT][2]) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    uint32_t most = 0;
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

// The records' rows from global memory, then w4_prepare_records.
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
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const bool have = row >= 0 && k < sh.myb;
#pragma unroll
      for (int i = 0; i < 8; ++i) b[k][j][i] = have ? __ldg(src + k * 32 + 4 * i) : 0u;
    }
  }
  w4_prepare_records<KB, NT, MODE>(b, fold, inv);
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

// Cuts a projection over the warps, kb blocks to each.
inline W4Plan w4_plan(const W4Matrix& m, int kb) {
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
inline int w4_best_kb(int nb, std::initializer_list<int> kbs) {
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

inline W4Matrix w4_matrix(const W4Bank& bank, bool down) {
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

}  // namespace moe
