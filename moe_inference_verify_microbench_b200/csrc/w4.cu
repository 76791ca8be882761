// Grouped products with 4-bit expert weights (layout: w4.cuh).
//
//   w4_stream<true>   h[p] = silu(A[p] . Wg[e]) * (A[p] . Wu[e]), A[p] =
//                     src[index[p] / index_div]
//   w4_stream<false>  out[row_map[p]] = row_scale[row_map[p]] * (h[p] . Wd[e])
//
// At few records per expert these are a stream of weights: 0.5 byte and the
// group's share of a scale per weight, so HBM bounds them and everything else
// has to stay below 23 bytes of weights per cycle and SM.  One persistent CTA per SM; a
// producer thread copies whole 16-row tiles (contiguous, with their scales) into a
// ring of shared-memory stages; eight consumer warps turn codes into bf16
// operands in registers (28 integer instructions per 1024 weights and warp, no
// conversion) and multiply them on the tensor cores as the 16-row operand of
// mma.m16n8k16, with up to 32 records as its columns.  The records' rows are
// held in registers for all tiles of an expert, so shared memory sees each
// weight once and no activation at all.  Up to eight warps share a tile along
// K and add their fp32 partials through shared memory.
//
// Numerics: products of bf16 activations with (q - z) are exact in fp32; each
// 64-column block (32 where the group is 32) is summed on the tensor cores in
// fp32 and then scaled in fp32, so no weight is ever rounded to bf16.
#include <algorithm>
#include <atomic>

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
  uint8_t* z;
  int* status;
};

__device__ __forceinline__ uint32_t w4_word(const uint8_t* codes, bool& bad) {
  const uint2 v = *reinterpret_cast<const uint2*>(codes);  // columns 0..3, 4..7
  bad |= ((v.x | v.y) & 0xf0f0f0f0u) != 0;
  uint32_t w = 0;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint32_t q = ((c < 4 ? v.x : v.y) >> (8 * (c & 3))) & 0xfu;
    w |= q << (4 * ((c >> 1) + 4 * (c & 1)));
  }
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
    const size_t col = static_cast<size_t>(kb) * 64 + 8 * t;
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
    a.s[2 * i] = a.scales[0][o0];
    a.s[2 * i + 1] = a.scales[pair ? 1 : 0][o1];
    if (a.z != nullptr) {
      const uint8_t z0 = a.zeros[0][o0], z1 = a.zeros[pair ? 1 : 0][o1];
      bad |= z0 > 15 || z1 > 15;
      a.z[2 * i] = z0 & 15;
      a.z[2 * i + 1] = z1 & 15;
    }
  }
  if (bad) record_status(a.status, kErrBadCode);
}

// ------------------------------------------------------------------ streaming

struct W4Args {
  W4Matrix m;
  W4Plan p;
  const uint4* act;     // A rows [act_rows][K]
  int act_rows;
  const int* index;     // A row of record p = act[index[p] / index_div] (null = p)
  int index_div;
  int M;                // records
  const int4* tiles;
  const int* num_tiles;
  int max_tiles;
  int E;
  __nv_bfloat16* out;
  int out_ld;
  int out_rows;
  const int* row_map;
  const float* row_scale;
  int* status;
};

// Work of a tile-table entry: its records in chunks of p.nr, each chunk one
// pass over the expert's stages (units).  A bad entry has none and is
// reported.
__device__ __forceinline__ int w4_units(const W4Args& a, const int4& t) {
  if (t.x < 0 || t.x >= a.E || t.y < 0 || t.z > a.M || t.z <= t.y) {
    if (t.z != t.y || t.x < 0 || t.x >= a.E)
      record_status(a.status, t.x < 0 || t.x >= a.E ? kErrBadExpert : kErrBadRow);
    return 0;
  }
  return (t.z - t.y + a.p.nr - 1) / a.p.nr * a.p.groups;
}

// Cost of a unit: the stream of its weights, and a share for every eight
// records multiplied with them.
__device__ __forceinline__ int w4_unit_cost(const W4Args& a, const int4& t) {
  return 6 + (min(t.z - t.y, a.p.nr) + 7) / 8;
}

struct W4Pos {
  int entry, unit;
};

// This CTA's contiguous range of units [lo, hi), the summed cost split evenly
// over the grid.  Every thread of the CTA calls it.
__device__ __forceinline__ void w4_range(const W4Args& a, int nt, W4Pos* lo, W4Pos* hi) {
  __shared__ long long sh_scan[32];
  __shared__ W4Pos sh_pos[2];
  __shared__ long long sh_total;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  auto cost = [&](int i) -> long long {
    if (i >= nt) return 0;
    const int4 t = a.tiles[i];
    const int u = w4_units(a, t);
    return u > 0 ? static_cast<long long>(u) * w4_unit_cost(a, t) : 0;
  };
  auto scan = [&](long long v, long long* total) {  // inclusive, over the block
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    if (lane == 31) sh_scan[warp] = v;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < nw; ++w) {
      const long long s = sh_scan[w];
      if (w < warp) before += s;
      all += s;
    }
    __syncthreads();
    *total = all;
    return before + v;
  };
  if (threadIdx.x == 0) {
    sh_pos[0] = sh_pos[1] = {0, 0};
    sh_total = 0;
  }
  long long total = 0;
  for (int base = 0; base < nt; base += blockDim.x) {
    long long part;
    scan(cost(base + static_cast<int>(threadIdx.x)), &part);
    total += part;
  }
  long long carry = 0;
  for (int base = 0; base < nt; base += blockDim.x) {
    const int i = base + static_cast<int>(threadIdx.x);
    const long long c = cost(i);
    long long part;
    const long long incl = scan(c, &part) + carry;
    carry += part;
    if (c > 0) {
      const int per = w4_unit_cost(a, a.tiles[i]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const long long want = total * (static_cast<long long>(blockIdx.x) + k) / gridDim.x;
        if (want > incl - c && want <= incl)
          sh_pos[k] = {i, static_cast<int>((want - (incl - c) + per - 1) / per)};
      }
    }
  }
  __syncthreads();
  *lo = sh_pos[0];
  *hi = sh_pos[1];
}

// The ring of stages in shared memory.
struct W4Ring {
  uint8_t* base;
  uint64_t* full;
  uint64_t* empty;
  volatile int* abort_flag;
  int s;
  uint32_t ph;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) {
      s = 0;
      ph ^= 1u;
    }
  }
};

// Copies tiles [tile0, tile0 + n) of expert e into the next stage (one thread).
__device__ __forceinline__ bool w4_produce(const W4Matrix& m, const W4Plan& p, W4Ring& r, int e,
                                           int tile0, int n, int* status) {
  if (!mbar_wait(&r.empty[r.s], r.ph ^ 1u, r.abort_flag, status, kErrTimeoutEmpty)) return false;
  const uint32_t qb = static_cast<uint32_t>(n) * m.nb * kW4BlockBytes;
  const uint32_t sb = static_cast<uint32_t>(n) * m.ng * 32, zb = m.z != nullptr ? sb / 2 : 0u;
  const size_t et = static_cast<size_t>(e) * m.tiles + tile0;
  uint8_t* dst = r.base + r.s * p.stage_bytes;
  mbar_arrive_expect_tx(&r.full[r.s], qb + sb + zb);
  bulk_load(dst, m.q + et * m.nb * kW4BlockBytes, qb, &r.full[r.s]);
  bulk_load(dst + p.s_off, m.s + et * m.ng * 32, sb, &r.full[r.s]);
  if (zb != 0) bulk_load(dst + p.z_off, m.z + et * m.ng * 16, zb, &r.full[r.s]);
  r.next(p.stages);
  return true;
}

// After an abort: every copy of the last `issued` stages lands before the CTA exits.
__device__ __forceinline__ void w4_drain(uint64_t* full, int stages, uint32_t issued) {
  const uint32_t n = static_cast<uint32_t>(stages);
  for (uint32_t i = issued > n ? issued - n : 0u; i < issued; ++i) {
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_wait(&full[i % n], (i / n) & 1u)) {
      if (globaltimer_ns() - t0 > kWaitLimitNs) break;
    }
  }
}

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ uint4 lds128(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(smem_u32(p))
               : "memory");
  return v;
}

__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// acc += scale * (codes of one 16 x 64 block - zero points) . records.
// FOLD (no zero points, group >= 64): the operand is 128 + q and the sum starts
// at -136 * (sum of the block's activations), `fold`, so the subtraction of
// 128 + 8 costs nothing; it cancels to within 2^-23 * 136 * sum|x| of the block.
// Otherwise 128 + z is subtracted from every operand, which is exact.
template <int NT, bool FOLD>
__device__ __forceinline__ void w4_block(float (&acc)[NT][4], const uint4& w,
                                         const uint32_t (&b)[NT][8], const float (&fold)[NT][2],
                                         const uint8_t* sp, const uint8_t* zp, int sg0, int sg1) {
  uint32_t z0[2] = {0x43084308u, 0x43084308u}, z1[2] = {0x43084308u, 0x43084308u};
  const uint32_t sc0 = *reinterpret_cast<const uint32_t*>(sp + sg0 * 32);
  uint32_t sc1 = sc0;
  if constexpr (!FOLD) {
    if (sg1 != sg0) sc1 = *reinterpret_cast<const uint32_t*>(sp + sg1 * 32);
    if (zp != nullptr) {
      const uint32_t v0 = *reinterpret_cast<const uint16_t*>(zp + sg0 * 16);
      const uint32_t v1 = *reinterpret_cast<const uint16_t*>(zp + sg1 * 16);
      z0[0] = (0x4300u | (v0 & 0xffu)) * 0x10001u;
      z0[1] = (0x4300u | (v0 >> 8)) * 0x10001u;
      z1[0] = (0x4300u | (v1 & 0xffu)) * 0x10001u;
      z1[1] = (0x4300u | (v1 >> 8)) * 0x10001u;
    }
  }
  float d[NT][4];
#pragma unroll
  for (int st = 0; st < 4; ++st) {
    const uint32_t wl = st < 2 ? w.x : w.y, wh = st < 2 ? w.z : w.w;
    const int i = 2 * (st & 1);
    uint32_t a[4] = {w4_pair(wl, i), w4_pair(wh, i), w4_pair(wl, i + 1), w4_pair(wh, i + 1)};
    if constexpr (!FOLD) {
      const uint32_t zl = st < 2 ? z0[0] : z1[0], zh = st < 2 ? z0[1] : z1[1];
      a[0] = sub_bf16x2(a[0], zl);
      a[1] = sub_bf16x2(a[1], zh);
      a[2] = sub_bf16x2(a[2], zl);
      a[3] = sub_bf16x2(a[3], zh);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (st == 0 || (!FOLD && st == 2 && sg1 != sg0)) {
        if (!FOLD && st == 2) {  // group 32: the first half is complete
#pragma unroll
          for (int c = 0; c < 4; ++c)
            acc[j][c] = fmaf(c < 2 ? bf16_lo(sc0) : bf16_hi(sc0), d[j][c], acc[j][c]);
        }
        float c0[4];
        c0[0] = c0[2] = FOLD ? fold[j][0] : 0.0f;
        c0[1] = c0[3] = FOLD ? fold[j][1] : 0.0f;
        mma_16816(d[j], a, b[j][2 * st], b[j][2 * st + 1], c0);
      } else {
        mma_16816(d[j], a, b[j][2 * st], b[j][2 * st + 1], d[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc[j][c] = fmaf(c < 2 ? bf16_lo(sc1) : bf16_hi(sc1), d[j][c], acc[j][c]);
}

// Record columns (in eights) a warp can hold next to KBT blocks: 128 registers
// of operands either way.
template <int KBT>
constexpr int w4_max_nt() {
  return KBT <= 4 ? 4 : KBT <= 8 ? 2 : 1;
}

// One record chunk's pass over units [u0, u1) of an entry (u counts stages
// within the chunk): records t.y + rec0 .. + n, n <= 8 NT.  Every consumer
// warp calls it; a warp whose wait gave up goes on without reading or storing, so the
// others never wait for it at a barrier.
template <bool SWIGLU, int KBT, int NT, bool FOLD>
__device__ __forceinline__ void w4_consume(const W4Args& a, W4Ring& r, float* part, uint32_t& round,
                                           int rec0, int n, int g0, int g1, bool& ok) {
  const W4Plan& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ks = warp % p.ks, tl = warp / p.ks;
  const int g = lane >> 2, t = lane & 3;
  const int kb0 = ks * p.kbn;
  const int myb = max(0, min(p.kbn, a.m.nb - kb0));
  const int vec = a.m.nb * 8;  // 16-byte vectors per A row
  uint32_t b[KBT][NT][8];
  float fold[KBT][NT][2];
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
    const uint4* src = a.act + static_cast<size_t>(max(row, 0)) * vec + kb0 * 8 + t;
#pragma unroll
    for (int k = 0; k < KBT; ++k) {
      uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0;
      if (row >= 0 && k < myb) {
        v0 = __ldg(src + k * 8);
        v1 = __ldg(src + k * 8 + 4);
      }
      b[k][j][0] = v0.x, b[k][j][1] = v0.y, b[k][j][2] = v0.z, b[k][j][3] = v0.w;
      b[k][j][4] = v1.x, b[k][j][5] = v1.y, b[k][j][6] = v1.z, b[k][j][7] = v1.w;
    }
  }
  if constexpr (FOLD) {
    // sums of a block's activations for this lane's columns, as a product with ones
    const uint32_t one[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
    for (int k = 0; k < KBT; ++k)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < 4; ++st) mma_16816(d, one, b[k][j][2 * st], b[k][j][2 * st + 1], d);
        fold[k][j][0] = -136.0f * d[0];
        fold[k][j][1] = -136.0f * d[1];
      }
  }
  for (int gi = g0; gi < g1; ++gi) {
    const int tile0 = gi * p.ts;
    const int nt = min(p.ts, a.m.tiles - tile0);
    if (ok && !mbar_wait(&r.full[r.s], r.ph, r.abort_flag, a.status, kErrTimeoutFull)) ok = false;
    ok = __all_sync(0xffffffffu, ok);
    const uint8_t* stage = r.base + r.s * p.stage_bytes;
    for (int tt = tl; tt < nt; tt += p.tl) {
      float acc[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
      const uint8_t* qp = stage + (tt * a.m.nb + kb0) * kW4BlockBytes + lane * 16;
      const uint8_t* sp = stage + p.s_off + tt * a.m.ng * 32 + g * 4;
      const uint8_t* zp = a.m.z != nullptr ? stage + p.z_off + tt * a.m.ng * 16 + g * 2 : nullptr;
      if (ok) {
#pragma unroll
        for (int k = 0; k < KBT; ++k) {
          if (k < myb) {
            const int half = 2 * (kb0 + k);
            w4_block<NT, FOLD>(acc, lds128(qp + k * kW4BlockBytes), b[k], fold[k], sp, zp,
                               half >> a.m.gshift, (half + 1) >> a.m.gshift);
          }
        }
      }
      if (p.ks > 1) {
        // partials of the ks warps: [buffer][warp][value][lane]
        constexpr int kStride = w4_max_nt<KBT>() * 128;  // the same for every NT
        float* pw = part + ((round & 1u) * kW4Warps + warp) * kStride + lane;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) pw[(4 * j + c) * 32] = acc[j][c];
        named_barrier(1 + tl, p.ks * 32);
        const float* pr = part + ((round & 1u) * kW4Warps + tl * p.ks) * kStride + lane;
#pragma unroll
        for (int u = 0; u < 2 * NT; ++u) {
          if ((u & (p.ks - 1)) == ks) {
            float s0 = 0.0f, s1 = 0.0f;
            for (int w = 0; w < p.ks; ++w) {
              s0 += pr[w * kStride + (4 * (u >> 1) + (u & 1)) * 32];
              s1 += pr[w * kStride + (4 * (u >> 1) + (u & 1) + 2) * 32];
            }
            acc[u >> 1][u & 1] = s0;
            acc[u >> 1][(u & 1) + 2] = s1;
          }
        }
        ++round;
      }
#pragma unroll
      for (int u = 0; u < 2 * NT; ++u) {
        const int rec = 8 * (u >> 1) + 2 * t + (u & 1);
        if ((u & (p.ks - 1)) == ks && rec < n && ok) {
          const float v0 = acc[u >> 1][u & 1], v1 = acc[u >> 1][(u & 1) + 2];
          const int tile = tile0 + tt;
          if constexpr (SWIGLU) {
            a.out[static_cast<size_t>(rec0 + rec) * a.out_ld + tile * 8 + g] =
                __float2bfloat16_rn(silu_f(v0) * v1);
          } else {
            const int o = a.row_map != nullptr ? __ldg(a.row_map + rec0 + rec) : rec0 + rec;
            if (o >= 0 && o < a.out_rows) {
              const float sc = a.row_scale != nullptr ? __ldg(a.row_scale + o) : 1.0f;
              __nv_bfloat16* dst = a.out + static_cast<size_t>(o) * a.out_ld + tile * 16 + g;
              dst[0] = __float2bfloat16_rn(v0 * sc);
              dst[8] = __float2bfloat16_rn(v1 * sc);
            } else {
              record_status(a.status, kErrBadRow);
            }
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0 && ok) mbar_arrive(&r.empty[r.s]);
    r.next(p.stages);
  }
}

template <int N>
__device__ __forceinline__ void setmaxnreg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void setmaxnreg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Units [lo, hi) of the tile table on this CTA: warp 8 produces, warps 0..7
// consume.
template <bool SWIGLU, int KBT, bool FOLD>
__device__ __forceinline__ void w4_units_loop(const W4Args& a, W4Ring r, float* part, int nt,
                                              W4Pos lo, W4Pos hi) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const W4Plan& p = a.p;
  constexpr int kMaxNT = w4_max_nt<KBT>();
  if (warp >= kW4Warps) {
    setmaxnreg_dec<kW4ProducerRegs>();
    if (warp != kW4Warps || lane != 0) return;
    uint32_t issued = 0;
    bool ok = true;
    for (int e = lo.entry; ok && e <= hi.entry && e < nt; ++e) {
      const int4 t = a.tiles[e];
      const int units = w4_units(a, t);
      const int u1 = e == hi.entry ? min(hi.unit, units) : units;
      for (int u = e == lo.entry ? lo.unit : 0; u < u1; ++u) {
        const int tile0 = u % p.groups * p.ts;
        if (!w4_produce(a.m, p, r, t.x, tile0, min(p.ts, a.m.tiles - tile0), a.status)) {
          ok = false;
          break;
        }
        ++issued;
      }
    }
    if (*r.abort_flag) w4_drain(r.full, p.stages, issued);
    return;
  }
  setmaxnreg_inc<kW4ConsumerRegs>();
  uint32_t round = 0;
  bool ok = true;
  for (int e = lo.entry; e <= hi.entry && e < nt; ++e) {
    const int4 t = a.tiles[e];
    const int units = w4_units(a, t);
    const int u1 = e == hi.entry ? min(hi.unit, units) : units;
    for (int u = e == lo.entry ? lo.unit : 0; u < u1;) {
      const int chunk = u / p.groups;
      const int g0 = u - chunk * p.groups;
      const int g1 = min(p.groups, g0 + u1 - u);
      const int rec0 = t.y + chunk * p.nr;
      const int n = min(p.nr, t.z - rec0);
      if (kMaxNT >= 4 && n > 16)
        w4_consume<SWIGLU, KBT, kMaxNT >= 4 ? 4 : 1, FOLD>(a, r, part, round, rec0, n, g0, g1, ok);
      else if (kMaxNT >= 2 && n > 8)
        w4_consume<SWIGLU, KBT, kMaxNT >= 2 ? 2 : 1, FOLD>(a, r, part, round, rec0, n, g0, g1, ok);
      else
        w4_consume<SWIGLU, KBT, 1, FOLD>(a, r, part, round, rec0, n, g0, g1, ok);
      u += g1 - g0;
    }
  }
}

template <int KBT>
constexpr int w4_part_bytes() {
  return 2 * kW4Warps * w4_max_nt<KBT>() * 128 * 4;
}
constexpr int kW4RingBytes = 184 * 1024;
constexpr int kW4TailBytes = 2 * kW4MaxStages * 8 + 16;

template <bool SWIGLU, int KBT, bool FOLD>
__global__ void __launch_bounds__(kW4Threads, 1) w4_stream(const W4Args a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint8_t* tail = smem_raw + kW4RingBytes + w4_part_bytes<KBT>();
  W4Ring r;
  r.base = smem_raw;
  r.full = reinterpret_cast<uint64_t*>(tail);
  r.empty = r.full + kW4MaxStages;
  r.abort_flag = reinterpret_cast<volatile int*>(r.empty + kW4MaxStages);
  r.s = 0;
  r.ph = 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < a.p.stages; ++s) {
      mbar_init(&r.full[s], 1);
      mbar_init(&r.empty[s], kW4Warps);
    }
    *r.abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int nt = max(0, min(*a.num_tiles, a.max_tiles));
  W4Pos lo, hi;
  w4_range(a, nt, &lo, &hi);
  w4_units_loop<SWIGLU, KBT, FOLD>(a, r, reinterpret_cast<float*>(smem_raw + kW4RingBytes), nt, lo,
                                   hi);
}

// ------------------------------------------------------------------ launchers

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class Kernel>
static bool allow_smem(Kernel* fn, int bytes, std::atomic<uint64_t>& done) {
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

// Cuts a projection over the warps: the fewest idle block slots, then the most
// warps to a tile (a shorter pass over a tile balances better over the SMs).
static W4Plan w4_plan(const W4Matrix& m) {
  W4Plan p{};
  long long best = -1;
  for (int ks = kW4Warps; ks >= 1; ks /= 2) {
    const int kbn = (m.nb + ks - 1) / ks;
    if (kbn > 16) break;
    const long long waste = static_cast<long long>(kbn) * ks - m.nb;
    if (best < 0 || waste * p.kbn * p.ks < best * kbn * ks) {
      // fewer warps to a tile only while the records still fit (kbn <= 4)
      if (best >= 0 && kbn > 4) break;
      best = waste;
      p.ks = ks;
      p.kbn = kbn;
    }
  }
  if (best < 0) return p;
  p.tl = kW4Warps / p.ks;
  const int tile_bytes = m.nb * kW4BlockBytes + m.ng * (m.z != nullptr ? 48 : 32);
  const int want = std::max(1, 12 * 1024 / (p.tl * tile_bytes));
  p.ts = p.tl * want;
  p.groups = (m.tiles + p.ts - 1) / p.ts;
  p.nr = 8 * (p.kbn <= 4 ? 4 : p.kbn <= 8 ? 2 : 1);
  p.s_off = p.ts * m.nb * kW4BlockBytes;
  p.z_off = p.s_off + p.ts * m.ng * 32;
  p.stage_bytes = (p.ts * tile_bytes + 127) / 128 * 128;
  p.stages = std::min(kW4MaxStages, kW4RingBytes / p.stage_bytes);
  return p;
}

static W4Matrix w4_matrix(const W4Bank& bank, bool down) {
  W4Matrix m{};
  m.q = static_cast<const uint8_t*>(down ? bank.w2_q : bank.w13_q);
  m.s = static_cast<const uint8_t*>(down ? bank.w2_s : bank.w13_s);
  m.z = static_cast<const uint8_t*>(down ? bank.w2_z : bank.w13_z);
  m.tiles = down ? bank.H / 16 : bank.I / 8;
  const int K = down ? bank.I : bank.H;
  m.nb = K / 64;
  m.ng = K / bank.group;
  m.gshift = bank.group == 32 ? 0 : bank.group == 64 ? 1 : 2;
  return m;
}

int w4_check_bank(const W4Bank& b) {
  if (b.E <= 0 || b.H <= 0 || b.I <= 0 || b.w13_q == nullptr || b.w13_s == nullptr ||
      b.w2_q == nullptr || b.w2_s == nullptr || (b.w13_z == nullptr) != (b.w2_z == nullptr))
    return kRcBadArgument;
  if (b.group != 32 && b.group != 64 && b.group != 128) return kRcUnsupported;
  if (b.H % 64 != 0 || b.I % 64 != 0 || b.H % b.group != 0 || b.I % b.group != 0 ||
      b.H > kW4MaxK || b.I > kW4MaxK || b.E > 1024)
    return kRcUnsupported;
  for (const void* p : {b.w13_q, b.w13_s, b.w13_z, b.w2_q, b.w2_s, b.w2_z})
    if (!aligned16(p)) return kRcBadArgument;
  return kRcOk;
}

template <bool SWIGLU, int KBT, bool FOLD>
static int w4_launch(const W4Args& a, cudaStream_t stream) {
  constexpr int sh = kW4RingBytes + w4_part_bytes<KBT>() + kW4TailBytes;
  static std::atomic<uint64_t> attr{0};
  if (!allow_smem(w4_stream<SWIGLU, KBT, FOLD>, sh, attr)) return kRcCudaError;
  const long long units = static_cast<long long>(a.max_tiles) * a.p.groups *
                          ((kBM + a.p.nr - 1) / a.p.nr);
  const int grid = static_cast<int>(std::min<long long>(units, device_sm_count()));
  return note_cuda_error(launch_pdl(w4_stream<SWIGLU, KBT, FOLD>, dim3(grid), dim3(kW4Threads), sh,
                                    stream, a)) == cudaSuccess
             ? kRcOk
             : kRcCudaError;
}

template <bool SWIGLU>
static int w4_dispatch(const W4Args& a, cudaStream_t stream) {
  const bool fold = a.m.z == nullptr && a.m.gshift > 0;
  if (a.p.kbn <= 4)
    return fold ? w4_launch<SWIGLU, 4, true>(a, stream) : w4_launch<SWIGLU, 4, false>(a, stream);
  if (a.p.kbn <= 8)
    return fold ? w4_launch<SWIGLU, 8, true>(a, stream) : w4_launch<SWIGLU, 8, false>(a, stream);
  return fold ? w4_launch<SWIGLU, 16, true>(a, stream) : w4_launch<SWIGLU, 16, false>(a, stream);
}

int launch_w4_w13(const W4Bank& bank, const void* src, int src_rows, const int* index,
                  int index_div, int M, const int4* tiles, const int* num_tiles, int max_tiles,
                  void* h_out, int* status, cudaStream_t stream) {
  if (const int rc = w4_check_bank(bank); rc != kRcOk) return rc;
  if (M < 0 || max_tiles < 0 || index_div <= 0 || src_rows < 0 || tiles == nullptr ||
      num_tiles == nullptr)
    return kRcBadArgument;
  if (M == 0 || max_tiles == 0) return kRcOk;
  if (src == nullptr || h_out == nullptr || !aligned16(src)) return kRcBadArgument;
  W4Args a{};
  a.m = w4_matrix(bank, false);
  a.p = w4_plan(a.m);
  a.act = static_cast<const uint4*>(src);
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
  a.status = status;
  return w4_dispatch<true>(a, stream);
}

int launch_w4_w2(const W4Bank& bank, const void* h, int M, const int4* tiles, const int* num_tiles,
                 int max_tiles, const int* row_map, const float* row_scale, void* out,
                 int out_rows, int* status, cudaStream_t stream) {
  if (const int rc = w4_check_bank(bank); rc != kRcOk) return rc;
  if (M < 0 || max_tiles < 0 || out_rows < 0 || tiles == nullptr || num_tiles == nullptr)
    return kRcBadArgument;
  if (M == 0 || max_tiles == 0) return kRcOk;
  if (h == nullptr || out == nullptr || !aligned16(h)) return kRcBadArgument;
  W4Args a{};
  a.m = w4_matrix(bank, true);
  a.p = w4_plan(a.m);
  a.act = static_cast<const uint4*>(h);
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
  a.status = status;
  return w4_dispatch<false>(a, stream);
}

int launch_w4_pack(const uint8_t* codes0, const void* scales0, const uint8_t* zeros0,
                   const uint8_t* codes1, const void* scales1, const uint8_t* zeros1, int E, int N,
                   int K, int group, void* q, void* s, void* z, int* status, cudaStream_t stream) {
  if (codes0 == nullptr || scales0 == nullptr || q == nullptr || s == nullptr ||
      (codes1 == nullptr) != (scales1 == nullptr) || (z == nullptr) != (zeros0 == nullptr) ||
      (codes1 != nullptr && (zeros0 == nullptr) != (zeros1 == nullptr)) ||
      (codes1 == nullptr && zeros1 != nullptr) || E <= 0 || N <= 0 || K <= 0)
    return kRcBadArgument;
  if ((group != 32 && group != 64 && group != 128) || K % 64 != 0 || K % group != 0 ||
      K > kW4MaxK || N % (codes1 != nullptr ? 8 : 16) != 0 || E > 1024)
    return kRcUnsupported;
  if (!aligned16(q) || !aligned16(s) || !aligned16(z) || !aligned16(codes0) || !aligned16(codes1))
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
  a.z = static_cast<uint8_t*>(z);
  a.status = status;
  return note_cuda_error(launch_pdl(w4_pack, dim3(device_sm_count() * 8), dim3(256), 0, stream,
                                    a)) == cudaSuccess
             ? kRcOk
             : kRcCudaError;
}

}  // namespace moe
