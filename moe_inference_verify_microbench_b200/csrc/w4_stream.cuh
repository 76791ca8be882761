// The streaming form of the grouped products with 4-bit weights: device code of the
// grouped kernels (w4.cu) and of the decode layer (w4_decode.cu).
#pragma once

#include <initializer_list>

#include "grouped_gemm.cuh"
#include "w4.cuh"

namespace moe {

// Work of a tile-table entry: its records in chunks of kW4Recs, each chunk one pass
// over the expert's tiles (units).  A bad entry has none and is reported.
__device__ __forceinline__ int w4_chunks(const W4Args& a, const int4& t) {
  if (!w4_entry_ok(a, t)) return 0;
  return (t.z - t.y + kW4Recs - 1) / kW4Recs;
}

// The contiguous range of units of one group of ks warps, the units split evenly
// over all groups of the grid, and a walk through it in runs of tiles that share
// their expert and records.  (Groups with ranges of their own load their
// records at different times: with the tiles of one range per CTA dealt out in turn,
// every group of the SM waited for its records at once.)
struct W4TableWalk {
  int entry, chunk, tile;  // next unit
  int chunks;              // of the entry
  int4 t;
  int nt, hi_entry, hi_unit;

  // Every thread of the CTA calls it.  The kernel serves tables of fewer than 8
  // records per expert on average, so 32 bits hold a table's units (2048 chunks x
  // 1024 tiles at most).
  __device__ __forceinline__ void open_range(const W4Args& a, int n_entries) {
    __shared__ uint32_t sums[kW4Warps];
    __shared__ int2 pos[kW4Warps + 1];
    nt = n_entries;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto units = [&](int i) -> uint32_t {
      return i < nt ? static_cast<uint32_t>(w4_chunks(a, a.tiles[i]) * a.m.tiles) : 0u;
    };
    const uint32_t first = units(threadIdx.x);  // most tables fit the CTA
    uint32_t mine = first;
    for (int i = threadIdx.x + kW4Threads; i < nt; i += kW4Threads) mine += units(i);
    if (threadIdx.x <= kW4Warps) pos[threadIdx.x] = make_int2(0, 0);
    uint32_t total = 0, carry = 0;
    for (int base = 0; base < nt; base += kW4Threads) {
      const uint32_t c = base == 0 ? first : units(base + static_cast<int>(threadIdx.x));
      uint32_t incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (base == 0) {  // the grand total, once
        const uint32_t all =
            nt <= kW4Threads ? __shfl_sync(0xffffffffu, incl, 31) : __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) sums[warp] = all;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kW4Warps; ++w) total += sums[w];
      }
      if (nt > kW4Threads) {
        __syncthreads();
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
      }
      uint32_t before = carry;
#pragma unroll
      for (int w = 0; w < kW4Warps; ++w) {
        const uint32_t s = sums[w];
        if (w < warp) before += s;
        carry += s;
      }
      incl += before;
      // the boundaries of this CTA's groups that fall into this entry
      const uint32_t parts = gridDim.x * a.p.tl;
      for (int k = 0; k <= a.p.tl; ++k) {
        const uint32_t want = static_cast<uint32_t>(
            static_cast<unsigned long long>(total) * (blockIdx.x * a.p.tl + k) / parts);
        if (want > incl - c && want <= incl)
          pos[k] = make_int2(base + static_cast<int>(threadIdx.x), static_cast<int>(want - (incl - c)));
      }
    }
    __syncthreads();
    const int tl = warp >> a.p.ks_shift;
    entry = pos[tl].x;
    tile = pos[tl].y;
    chunk = 0;
    hi_entry = pos[tl + 1].x;
    hi_unit = pos[tl + 1].y;
    open(a);
  }
  __device__ __forceinline__ void open(const W4Args& a) {
    for (chunks = 0; entry < nt; ++entry) {
      t = a.tiles[entry];
      chunks = w4_chunks(a, t);
      if (chunks > 0) return;
    }
  }
  __device__ __forceinline__ int expert() const { return t.x; }
  __device__ __forceinline__ int first() const { return t.y + chunk * kW4Recs; }
  __device__ __forceinline__ int count() const { return min(kW4Recs, t.z - first()); }
  // Tiles of the run that starts at the next unit: 0 at the end of the range.
  __device__ __forceinline__ int run(const W4Args& a) {
    while (tile >= a.m.tiles && entry < nt) {
      tile -= a.m.tiles;
      if (++chunk >= chunks) {
        chunk = 0;
        ++entry;
        open(a);
      }
    }
    if (entry >= nt || entry > hi_entry) return 0;
    const int end = entry == hi_entry ? min(a.m.tiles, hi_unit - chunk * a.m.tiles) : a.m.tiles;
    return max(end - tile, 0);
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
// 16-column steps.  With ZERO the zero points come off the operands first: z
// holds 128 + z of rows g and g + 8 in the halves.
template <bool ZERO>
__device__ __forceinline__ void w4_half(float (&d)[4], uint32_t wl, uint32_t wh, int h,
                                        const uint32_t (&b)[8], uint32_t z) {
  uint32_t lo[4], hi[4];
  w4_pairs(wl, lo);
  w4_pairs(wh, hi);
  if constexpr (ZERO) {
    const uint32_t zl = __byte_perm(z, 0, 0x1010), zh = __byte_perm(z, 0, 0x3232);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = sub_bf16x2(lo[i], zl);
      hi[i] = sub_bf16x2(hi[i], zh);
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s)
    mma_16816(d, lo[2 * s], hi[2 * s], lo[2 * s + 1], hi[2 * s + 1], b[4 * h + 2 * s],
              b[4 * h + 2 * s + 1]);
}

// acc += scale * d: the end of a group (or of the warp's share of it).
__device__ __forceinline__ void w4_flush(float (&acc)[4], const float (&d)[4], uint32_t sc) {
#pragma unroll
  for (int c = 0; c < 4; ++c) acc[c] = fmaf(c < 2 ? bf16_lo(sc) : bf16_hi(sc), d[c], acc[c]);
}

// What of a tile is this warp's.
struct W4Share {
  int ks, tl;    // its place along K, its place among the tiles worked on at once
  int kb0, myb;  // its blocks
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
  return s;
}

// Without zero points the weight operand stays 128 + q, and a group's sum starts
// at -136 times its activations (`fold`, kept at the group's first block), so the
// subtraction of 128 + 8 costs nothing per weight; it cancels to within 2^-23 *
// 136 * sum|x|.  kW4Half subtracts from every operand instead, which is exact.
// Every lane gets the sums of its columns from a product with the operand -136.
template <int KB, int MODE>
__device__ __forceinline__ void w4_fold(const uint32_t (&b)[KB][8], float (&fold)[KB][2]) {
  if constexpr (MODE != kW4Half) {
    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = KB - 1; k >= 0; --k) {
      if (MODE == kW4Block || (k & 1)) d[0] = d[1] = d[2] = d[3] = 0.0f;
#pragma unroll
      for (int st = 0; st < 4; ++st)
        mma_16816(d, 0xc308c308u, 0xc308c308u, 0xc308c308u, 0xc308c308u, b[k][2 * st],
                  b[k][2 * st + 1]);
      fold[k][0] = d[0];
      fold[k][1] = d[1];
    }
  }
}

// acc = this warp's share of a tile (its codes at `slot`, its group records at
// slot + KB blocks) times the records.
template <int KB, int MODE>
__device__ __forceinline__ void w4_tile(const W4Args& a, uint32_t slot, const uint32_t (&b)[KB][8],
                                        const float (&fold)[KB][2], float (&acc)[4]) {
  const int lane = threadIdx.x & 31;
  const uint32_t qp = slot + lane * 16;
  const uint32_t rec = slot + KB * kW4BlockBytes + (lane >> 2) * a.m.rec;
  const uint32_t step = 8 * a.m.rec;
  float d[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) acc[c] = 0.0f;
#pragma unroll
  for (int k = 0; k < KB; ++k) {
    const uint4 w = lds128(qp + k * kW4BlockBytes);
    if (MODE != kW4TwoBlocks || (k & 1) == 0) {
#pragma unroll
      for (int c = 0; c < 4; ++c) d[c] = MODE != kW4Half ? fold[k][c & 1] : 0.0f;
    }
    if constexpr (MODE != kW4Half) {
      w4_half<false>(d, w.x, w.z, 0, b[k], 0u);
      w4_half<false>(d, w.y, w.w, 1, b[k], 0u);
      if (MODE == kW4TwoBlocks && (k & 1)) w4_flush(acc, d, lds32(rec + (k >> 1) * (8 * 4)));
      if (MODE == kW4Block) w4_flush(acc, d, lds32(rec + k * (8 * 4)));
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t r = rec + ((2 * k + h) >> a.m.gshift) * step;
        const uint32_t z = a.m.rec == 8 ? lds32(r + 4) : 0x43084308u;
        w4_half<true>(d, h == 0 ? w.x : w.y, h == 0 ? w.z : w.w, h, b[k], z);
        w4_flush(acc, d, lds32(r));
        if (h == 0) d[0] = d[1] = d[2] = d[3] = 0.0f;
      }
    }
  }
}

// What a lane copies of every tile: its 16 bytes of each block, and a record of
// four groups at a time.  Blocks past the last are left as they are (any code times zero
// is zero), but every record that is read is a real one.
template <int KB, int MODE>
struct W4Lane {
  static constexpr int kSteps =  // of four groups
      MODE == kW4TwoBlocks ? (KB / 2 + 3) / 4 : MODE == kW4Block ? (KB + 3) / 4 : KB / 2;
  int from[kSteps];  // of the records, from the tile's first
  __device__ __forceinline__ W4Lane(const W4Args& a, const W4Share& sh) {
    const int lane = threadIdx.x & 31;
    const int g0 = (2 * sh.kb0) >> a.m.gshift;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      from[i] = (min(g0 + 4 * i + (lane >> 3), a.m.ng - 1) * 8 + (lane & 7)) * a.m.rec;
  }
  // Copies this warp's share of tile et (expert * tiles + tile) into a slot, asynchronously.
  __device__ __forceinline__ void fetch(const W4Args& a, const W4Share& sh, uint32_t slot,
                                        const uint8_t* q, const uint8_t* s) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < KB; ++k)
      if (k < sh.myb) cp_async_16(slot + lane * 16 + k * kW4BlockBytes, q + k * kW4BlockBytes, 16);
    const int groups = MODE == kW4TwoBlocks ? KB / 2 : MODE == kW4Block ? KB : (2 * KB) >> a.m.gshift;
    const uint32_t dst = slot + KB * kW4BlockBytes + lane * a.m.rec;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (4 * i + (lane >> 3) < groups) {
        if (MODE == kW4Half && a.m.rec == 8) cp_async_small<8>(dst + i * 256, s + from[i]);
        else cp_async_small<4>(dst + i * 128, s + from[i]);
      }
    }
  }
};

constexpr int kW4PartBytes = 2 * kW4Warps * 128 * 4;
constexpr int kW4SmemBytes = 224 * 1024;
template <int KB, int MODE>
constexpr int w4_slots() {
  return KB == 8 ? (MODE == kW4Half ? 2 : 3) : KB == 6 ? 3 : 4;
}

// The ks partials of a tile meet in shared memory: [buffer][warp][value][lane], two
// buffers so that one barrier per tile suffices.  Afterwards the value pairs
// u = 0, 1 (of records 2t + u) that this warp has, u modulo ks, are sums.
__device__ __forceinline__ void w4_meet(const W4Args& a, const W4Share& sh, float (&acc)[4],
                                        float* part, int buffer) {
  const W4Plan& p = a.p;
  if (p.ks == 1) return;
  const int lane = threadIdx.x & 31;
  float* pw = part + buffer + (sh.tl * p.ks + sh.ks) * 128 + lane;
#pragma unroll
  for (int v = 0; v < 4; ++v) pw[v * 32] = acc[v];
  named_barrier(1 + sh.tl, p.ks * 32);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if ((u & (p.ks - 1)) == sh.ks) {
      const float* pr = part + buffer + sh.tl * p.ks * 128 + u * 32 + lane;
      float v0 = 0.0f, v1 = 0.0f;
      for (int w = 0; w < p.ks; w += 2) {
        v0 += pr[0] + pr[128];
        v1 += pr[64] + pr[192];
        pr += 256;
      }
      acc[u] = v0;
      acc[u + 2] = v1;
    }
  }
}

// The units of a group's walk (copied for the fetches that run ahead of the
// products).
template <bool SWIGLU, int KB, int MODE, class Walk>
__device__ __forceinline__ void w4_units(const W4Args& a, uint8_t* smem, float* part, Walk c) {
  constexpr int SLOTS = w4_slots<KB, MODE>();
  const W4Plan& p = a.p;
  const W4Share sh = w4_share<KB>(a);
  const W4Lane<KB, MODE> own(a, sh);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t base = smem_u32(smem) + (sh.tl * p.ks + sh.ks) * SLOTS * p.slot_bytes;
  Walk f = c;                   // the next run to fetch; c: the run to work on
  const uint8_t* fq = nullptr;  // next tile to fetch
  const uint8_t* fs = nullptr;
  int left = f.run(a);
  uint32_t fslot = base, slot = base;
  const uint32_t end_slot = base + SLOTS * p.slot_bytes;
  const int q_tile = a.m.nb * kW4BlockBytes, s_tile = a.m.ng * 8 * a.m.rec;
  auto aim = [&]() {  // pointers of the run's first tile
    const size_t et = static_cast<size_t>(f.expert()) * a.m.tiles + f.tile;
    fq = a.m.q + et * q_tile + sh.kb0 * kW4BlockBytes + lane * 16;
    fs = a.m.s + et * s_tile;
  };
  if (left > 0) aim();
  auto fetch = [&]() {
    if (left > 0) {
      own.fetch(a, sh, fslot, fq, fs);
      fq += q_tile;
      fs += s_tile;
      ++f.tile;
      if (--left == 0) {
        left = f.run(a);
        if (left > 0) aim();
      }
    }
    cp_async_commit();
    fslot += p.slot_bytes;
    if (fslot == end_slot) fslot = base;
  };
#pragma unroll
  for (int i = 0; i < SLOTS - 1; ++i) fetch();
  int buffer = 0;
  for (int count; (count = c.run(a)) > 0;) {
    const int rec0 = c.first(), n = c.count();
    uint32_t b[KB][8];  // the records' rows: zeros past the last record and block
    {
      int row = -1;
      if (g < n) {
        row = a.index != nullptr ? a.index[rec0 + g] / a.index_div : rec0 + g;
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
        for (int i = 0; i < 8; ++i) b[k][i] = have ? __ldg(src + k * 32 + 4 * i) : 0u;
      }
    }
    // Value pairs u (records 2t + u) are stored by the warps u modulo ks: their
    // rows (-1: none) and scales.
    int orow[2];
    float scale[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int rec = 2 * t + u;
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
    float fold[KB][2];
    w4_fold<KB, MODE>(b, fold);
    int col = c.tile * (SWIGLU ? 8 : 16) + g;
    for (int i = 0; i < count; ++i) {
      cp_async_wait_group<SLOTS - 2>();
      __syncwarp();  // every lane's copies have landed, and the last tile's slot is free
      fetch();
      float acc[4];
      w4_tile<KB, MODE>(a, slot, b, fold, acc);
      slot += p.slot_bytes;
      if (slot == end_slot) slot = base;
      w4_meet(a, sh, acc, part, buffer);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (orow[u] >= 0) {
          const size_t at = static_cast<size_t>(orow[u]) * a.out_ld + col;
          if constexpr (SWIGLU) {
            a.out[at] = __float2bfloat16_rn(silu_f(acc[u]) * acc[u + 2]);
          } else if (a.out_f32 != nullptr) {
            a.out_f32[at] = acc[u] * scale[u];
            a.out_f32[at + 8] = acc[u + 2] * scale[u];
          } else {
            a.out[at] = __float2bfloat16_rn(acc[u] * scale[u]);
            a.out[at + 8] = __float2bfloat16_rn(acc[u + 2] * scale[u]);
          }
        }
      }
      col += SWIGLU ? 8 : 16;
      buffer ^= kW4Warps * 128;
    }
    c.tile += count;
  }
  cp_async_wait_all();  // nothing is in flight when the CTA exits
}

// Cuts a projection over the warps, kb blocks to each.
inline W4Plan w4_plan(const W4Matrix& m, int kb) {
  W4Plan p{};
  p.ks = 1;
  while (p.ks * kb < m.nb) p.ks *= 2;
  p.tl = kW4Warps / p.ks;
  while ((1 << p.ks_shift) < p.ks) ++p.ks_shift;
  const int groups = (2 * kb) >> m.gshift;  // kb is even: a share starts with a group
  p.slot_bytes = kb * kW4BlockBytes + groups * 8 * m.rec;
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
