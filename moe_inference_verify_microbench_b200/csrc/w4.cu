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
// codes into bf16 operands 128 + q in registers (seven integer instructions for
// eight weights, no conversion) and multiplies them on the tensor cores as the
// 16-row operand of mma.m16n8k16, with up to 8 records as its columns (more records
// of an expert: another pass).  The records' rows stay in registers for all tiles
// of an expert.  The warps that share a tile along K add their fp32 partials
// through shared memory.
//
// Measured back to back, 128 experts of 2048 x 768, top 8, group 128: gate/up 3.5
// TB/s at 12 tokens (30 us), 3.9 at 64 (52 us); down 2.6 and 3.2 TB/s.  The integer
// pipe is the next bound: it takes the extraction at half rate and is half busy (48 % of
// the issue slots, 66 instructions per 16 x 64 block); a shift of the seven done by
// mul.hi instead costs 3 us of 42.
//
// Numerics: products of activations with (q - z) are exact in fp32; each
// group (or a warp's share of it) is summed on the tensor cores in fp32 and
// then scaled in fp32, so no weight is ever rounded to bf16.
#include <cuda_fp16.h>

#include <algorithm>

#include "grouped_gemm.cuh"
#include "internal.h"
#include "w4_stream.cuh"

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
      rec[2] = 0x4300u | (z0 & 15u);  // bf16 128 + z
      rec[3] = 0x4300u | (z1 & 15u);
    }
  }
  if (bad) record_status(a.status, kErrBadCode);
}

// The records of the tensor-memory form, of the same shape: scales as fp16 multiples of a
// power of two, zero points as 1024 + z.  The power is the expert's, and puts its largest
// scale into [2^10, 2^11), so that fifteen times it is in fp16's range.  A bf16 scale has
// eight bits and stays exact down to 2^-17 (2^-27 of the largest); a row all of whose
// scales are below 2^-16 of the largest has a power of its own.  r[expert][tile][16] holds
// 1, or what such a row's power is of the expert's, and behind it, r[E * M + expert], the
// experts'.  A row with an infinity or a NaN keeps its scales.  blockIdx.x is the expert;
// its CTAs find its largest scale each for itself and share its rows.
__global__ void __launch_bounds__(256) w4_pack_fine(const W4PackArgs a, float* r) {
  pdl_wait();
  pdl_trigger();
  __shared__ int most;
  const int ng = a.K / a.group, e = blockIdx.x;
  const bool pair = a.scales[1] != nullptr;
  const int tiles = a.N / (pair ? 8 : 16);
  const bool zp = a.zeros[0] != nullptr;
  const size_t row0 = static_cast<size_t>(e) * a.N;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  int top = 0;
  for (int m = 0; m < (pair ? 2 : 1); ++m)
#pragma unroll 8
    for (int i = threadIdx.x; i < a.N * ng; i += blockDim.x) {
      const int v = a.scales[m][row0 * ng + i] & 0x7fff;
      if (v < 0x7f80) top = max(top, v);
    }
  atomicMax(&most, top);
  __syncthreads();
  auto shift_of = [](int bits) {
    return bits == 0 ? 0 : 10 - ilogbf(__uint_as_float(static_cast<uint32_t>(bits) << 16));
  };
  const int base = shift_of(most);
  if (threadIdx.x == 0 && blockIdx.y == 0)
    r[static_cast<size_t>(a.E) * tiles * 16 + e] = ldexpf(1.0f, -base);
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < tiles * 16; i += gridDim.y * blockDim.x) {
    const int tile = i >> 4, g = i & 7, half = (i >> 3) & 1;  // packed row g, or g + 8
    const int m = pair ? half : 0;
    const size_t row = row0 + (pair ? 8 * tile : 16 * tile + 8 * half) + g;
    const uint16_t* s = a.scales[m] + row * ng;
    top = 0;
    for (int k = 0; k < ng; ++k) top = max(top, s[k] & 0x7fff);
    int shift = base;
    if (top >= 0x7f80) shift = 0;
    else if (top > 0 && shift_of(top) - base > 16) shift = shift_of(top);
    const size_t et = static_cast<size_t>(e) * tiles + tile;
    r[et * 16 + (i & 15)] = top < 0x7f80 ? ldexpf(1.0f, base - shift) : 1.0f;
    uint16_t* out = a.s + (et * ng * 8 + g) * (zp ? 4 : 2) + half;
    for (int k = 0; k < ng; ++k, out += 8 * (zp ? 4 : 2)) {
      const float v = __uint_as_float(static_cast<uint32_t>(s[k]) << 16);
      out[0] = __half_as_ushort(__float2half_rn(ldexpf(v, shift)));
      if (zp) out[2] = 0x6400u | (a.zeros[m][row * ng + k] & 15u);
    }
  }
}

// ------------------------------------------------------------------ streaming

template <bool SWIGLU, int KB, int MODE>
__global__ void __launch_bounds__(kW4Threads, 1) w4_stream(const W4Args a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  pdl_wait();
  pdl_trigger();
  const int nt = max(0, min(*a.num_tiles, a.max_tiles));
  W4TableWalk walk;
  walk.open_range(a, nt);
  if constexpr (!SWIGLU) w4_zero_rest(a, nt, threadIdx.x, kW4Threads);
  w4_units<SWIGLU, KB, MODE>(a, smem_raw + kW4PartBytes, reinterpret_cast<float*>(smem_raw), walk);
}

// ------------------------------------------------------------------ launchers

int w4_check_bank(const W4Bank& b) {
  if (b.E <= 0 || b.H <= 0 || b.I <= 0 || b.w13_q == nullptr || b.w13_s == nullptr ||
      b.w2_q == nullptr || b.w2_s == nullptr)
    return kRcBadArgument;
  if (b.group != 32 && b.group != 64 && b.group != 128) return kRcUnsupported;
  if (b.H % 64 != 0 || b.I % 64 != 0 || b.H % b.group != 0 || b.I % b.group != 0 ||
      b.H > kW4MaxK || b.I > kW4MaxK || b.E > 1024)
    return kRcUnsupported;
  for (const void* p : {b.w13_q, b.w13_s, b.w2_q, b.w2_s, b.w13_f, b.w2_f,
                        static_cast<const void*>(b.w13_r), static_cast<const void*>(b.w2_r)})
    if (!aligned16(p)) return kRcBadArgument;
  const bool fine = b.w13_f != nullptr;
  if ((b.w2_f != nullptr) != fine || (b.w13_r != nullptr) != fine || (b.w2_r != nullptr) != fine)
    return kRcBadArgument;
  return kRcOk;
}

template <bool SWIGLU, int KB, int MODE>
static int w4_launch(W4Args& a, cudaStream_t stream) {
  a.p = w4_plan(a.m, KB);
  const int sh = kW4PartBytes + kW4Warps * w4_slots<KB, MODE>() * a.p.slot_bytes;
  if (sh > kW4SmemBytes) return kRcUnsupported;
  static std::atomic<uint64_t> attr{0};
  if (!allow_smem(w4_stream<SWIGLU, KB, MODE>, kW4SmemBytes, attr)) return kRcCudaError;
  const long long units = static_cast<long long>(a.max_tiles) * a.m.tiles;
  // a table of ranges that do not overlap has at most M / 8 chunks and one more an entry
  if (units + static_cast<long long>(a.M / kW4Recs) * a.m.tiles > 0xffffffffLL)
    return kRcUnsupported;  // the walk counts in 32 bits
  const int grid = static_cast<int>(std::min<long long>(units, device_sm_count()));
  return note_cuda_error(launch_pdl(w4_stream<SWIGLU, KB, MODE>, dim3(grid), dim3(kW4Threads), sh,
                                    stream, a)) == cudaSuccess
             ? kRcOk
             : kRcCudaError;
}

template <bool SWIGLU, int MODE>
static int w4_dispatch_mode(W4Args& a, cudaStream_t stream) {
  switch (w4_best_kb(a.m.nb, {4, 6, 8})) {
    case 4: return w4_launch<SWIGLU, 4, MODE>(a, stream);
    case 6: return w4_launch<SWIGLU, 6, MODE>(a, stream);
    case 8: return w4_launch<SWIGLU, 8, MODE>(a, stream);
  }
  return kRcUnsupported;
}

template <bool SWIGLU>
static int w4_dispatch(W4Args& a, cudaStream_t stream) {
  if (a.m.rec == 8 || a.m.gshift == 0) return w4_dispatch_mode<SWIGLU, kW4Half>(a, stream);
  if (a.m.gshift == 1) return w4_dispatch_mode<SWIGLU, kW4Block>(a, stream);
  return w4_dispatch_mode<SWIGLU, kW4TwoBlocks>(a, stream);
}

int launch_w4_w13(const W4Bank& bank, const void* src, int src_rows, const int* index,
                  int index_div, int M, const int4* tiles, const int* num_tiles, int max_tiles,
                  void* h_out, int avg, int* status, cudaStream_t stream, const W4Rows& rows,
                  float* h_f32) {
  if (const int rc = w4_check_bank(bank); rc != kRcOk) return rc;
  const bool many = w4_many(bank, avg) && rows.f16 != nullptr;
  if (M < 0 || max_tiles < 0 || index_div <= 0 || src_rows < 0 || tiles == nullptr ||
      num_tiles == nullptr)
    return kRcBadArgument;
  if (M == 0 || max_tiles == 0) return kRcOk;
  if (src == nullptr || src_rows == 0 || (h_out == nullptr) == (h_f32 == nullptr) ||
      !aligned16(src) || !aligned16(h_out) || !aligned16(h_f32) || !aligned16(tiles) ||
      (h_f32 != nullptr && !many))
    return kRcBadArgument;
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
  a.out_f32 = h_f32;
  a.out_ld = bank.I;
  a.out_rows = M;
  a.status = status;
  if (many) {
    a.m.s = static_cast<const uint8_t*>(bank.w13_f);
    a.row_factor = bank.w13_r;
    return w4_gemm(a, true, rows, false, stream);
  }
  return w4_dispatch<true>(a, stream);
}

int launch_w4_w2(const W4Bank& bank, const void* h, int M, const int4* tiles, const int* num_tiles,
                 int max_tiles, const int* row_map, const float* row_scale, void* out,
                 int out_rows, int avg, int* status, cudaStream_t stream, const W4Rows& rows,
                 bool zero_rest, float* out_f32, bool h_f32) {
  if (const int rc = w4_check_bank(bank); rc != kRcOk) return rc;
  const bool many = w4_many(bank, avg) && (rows.f16 != nullptr || h_f32);
  if (M < 0 || max_tiles < 0 || out_rows < 0 || tiles == nullptr || num_tiles == nullptr)
    return kRcBadArgument;
  if (M == 0 || max_tiles == 0) return kRcOk;
  if (h == nullptr || (out == nullptr) == (out_f32 == nullptr) || !aligned16(h) ||
      !aligned16(out) || !aligned16(tiles) || (out_f32 != nullptr && (zero_rest || many)) ||
      (h_f32 && !many))
    return kRcBadArgument;
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
  a.out_f32 = out_f32;
  a.out_ld = bank.H;
  a.out_rows = out_rows;
  a.row_map = row_map;
  a.row_scale = row_scale;
  a.zero_rest = zero_rest;
  a.status = status;
  if (many) {
    a.m.s = static_cast<const uint8_t*>(bank.w2_f);
    a.row_factor = bank.w2_r;
    return w4_gemm(a, false, rows, h_f32, stream);
  }
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

int launch_w4_pack_fine(const void* scales0, const uint8_t* zeros0, const void* scales1,
                        const uint8_t* zeros1, int E, int N, int K, int group, void* f, float* r,
                        cudaStream_t stream) {
  if (scales0 == nullptr || f == nullptr || r == nullptr || E <= 0 || N <= 0 || K <= 0 ||
      (scales1 != nullptr && (zeros0 == nullptr) != (zeros1 == nullptr)) ||
      (scales1 == nullptr && zeros1 != nullptr) || !aligned16(f) || !aligned16(r))
    return kRcBadArgument;
  if ((group != 32 && group != 64 && group != 128) || K % 64 != 0 || K % group != 0 ||
      K > kW4MaxK || N % (scales1 != nullptr ? 8 : 16) != 0 || E > 1024)
    return kRcUnsupported;
  W4PackArgs a{};
  a.scales[0] = static_cast<const uint16_t*>(scales0);
  a.scales[1] = static_cast<const uint16_t*>(scales1);
  a.zeros[0] = zeros0;
  a.zeros[1] = zeros1;
  a.E = E;
  a.N = N;
  a.K = K;
  a.group = group;
  a.s = static_cast<uint16_t*>(f);
  return note_cuda_error(launch_pdl(w4_pack_fine, dim3(E, std::max(1, 4 * device_sm_count() / E)),
                                    dim3(256), 0, stream, a, r)) == cudaSuccess
             ? kRcOk
             : kRcCudaError;
}

}  // namespace moe
