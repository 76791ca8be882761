// The whole mixture-of-experts layer for a few tokens on a 4-bit bank (T <= 16,
// T * k <= 64 records), in two kernels:
//
//   w4_logits  one warp per (token, expert): the router's logit, rounded to bf16 as
//              the router defines it; zeroes the layer's barrier counter
//   w4_layer   cooperative, one CTA of sixteen warps per SM:
//     1  every CTA takes the top-k of every token and sorts the records by expert
//     2  gate/up + SwiGLU over all CTAs as w4_stream<true>, h to the workspace
//     -  grid barrier; the first down weights are on their way before it
//     3  down: each CTA owns 16 rows of the output, for every routed expert, so
//        the weighted sum of a token's experts is its own: no slot rows, no second
//        barrier, no combine
//
// At one token this is a chain of latencies: 12.6 MB of gate and up codes and 6.3
// MB of down codes take 3 us of HBM time.  So every phase asks for all it will
// read at once: a warp has two tiles of codes in flight before it waits, and the
// down phase has one tile for each expert and warp group.
#include <algorithm>

#include "decode_route.cuh"
#include "w4_stream.cuh"

namespace moe {

namespace {

struct W4LayerArgs {
  W4Args up, down;  // tile tables and records are the kernel's own
  const uint4* x;   // [T][H]
  int T, k, E, norm_topk_prob;
  const float* logits;  // [T][E]
  unsigned int* bar;
  __nv_bfloat16* y;  // [T][H]
};

__global__ void __launch_bounds__(32) w4_logits(const uint4* __restrict__ x,
                                                const uint4* __restrict__ wr,
                                                const float* __restrict__ bias, int vec, int E,
                                                float* __restrict__ logits, unsigned int* bar) {
  constexpr int kEarly = 8;  // vectors of both rows asked for at once
  const int e = blockIdx.x % E, t = blockIdx.x / E, lane = threadIdx.x;
  const uint4* row = wr + static_cast<size_t>(e) * vec;
  pdl_wait();  // the weights too may have been written by the kernel before
  pdl_trigger();
  if (blockIdx.x == 0 && lane == 0) *bar = 0;
  const uint4* xr = x + static_cast<size_t>(t) * vec;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // the order of router_sort_small
  uint4 wv[kEarly], xv[kEarly];
#pragma unroll
  for (int j = 0; j < kEarly; ++j) {
    const int v = lane + 32 * j;
    wv[j] = v < vec ? __ldg(row + v) : make_uint4(0, 0, 0, 0);
    xv[j] = v < vec ? __ldg(xr + v) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < kEarly; ++j)
    if (lane + 32 * j < vec) dot8_acc(wv[j], xv[j], acc);
#pragma unroll 4
  for (int v = lane + 32 * kEarly; v < vec; v += 32) dot8_acc(__ldg(row + v), __ldg(xr + v), acc);
  const float sum = warp_sum(acc_sum(acc));
  if (lane == 0) logits[t * E + e] = bf16_round_f(sum + (bias != nullptr ? bias[e] : 0.0f));
}

constexpr int kLayerSmemBytes = 223 * 1024;  // beside 3.4 KB of static shared memory
constexpr int kLayerSlots = 2;   // of a warp in the down phase
constexpr int kLayerMaxT = 16;   // as the small router's
constexpr int kDsumBytes = kFusedMaxRecs * 16 * 4;

// Bytes between the staged rows of h: 16 more than a row, so that the eight rows
// of an operand start in different banks.
__host__ __device__ constexpr int h_pitch(int I) { return 2 * I + 16; }

// Down projection and weighted sum (phase 3).  Items are (expert tile, up to eight
// records); the groups of ks warps take them in turn.
template <int KB, int MODE>
__device__ __forceinline__ void w4_down(const W4LayerArgs& d, const RouteSmem& rs, uint8_t* smem,
                                        const int4* items, int nitems,
                                        volatile int* abort_flag) {
  const W4Args& a = d.down;
  const W4Plan& p = a.p;
  const W4Share sh = w4_share<KB>(a);
  const W4Lane<KB, MODE> own(a, sh);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warp = sh.tl * p.ks + sh.ks;
  float* part = reinterpret_cast<float*>(smem);
  uint8_t* slots = smem + kW4PartBytes;
  // the products of every record for a row tile, then the staged rows of h
  auto* dsum = reinterpret_cast<float(*)[16]>(slots + kW4Warps * kLayerSlots * p.slot_bytes);
  uint8_t* hs = reinterpret_cast<uint8_t*>(dsum + kFusedMaxRecs);
  const uint32_t base = smem_u32(slots) + warp * kLayerSlots * p.slot_bytes;
  const int pitch = h_pitch(64 * a.m.nb), R = d.T * d.k;
  const int grid = gridDim.x;

  // (row tile, item) to fetch next: this group's items of a row tile, then the next one's
  int f_tile = blockIdx.x, f_item = sh.tl, f_slot = 0;
  auto fetch = [&]() {
    if (f_tile < a.m.tiles && sh.tl < nitems) {
      const size_t et = static_cast<size_t>(items[f_item].x) * a.m.tiles + f_tile;
      own.fetch(a, sh, base + f_slot * p.slot_bytes,
                a.m.q + (et * a.m.nb + sh.kb0) * kW4BlockBytes + lane * 16,
                a.m.s + et * a.m.ng * 8 * a.m.rec);
      f_item += p.tl;
      if (f_item >= nitems) {
        f_item = sh.tl;
        f_tile += grid;
      }
    }
    cp_async_commit();
    f_slot ^= 1;
  };
  static_assert(kLayerSlots == 2, "f_slot alternates");
  fetch();  // the first codes do not depend on h: in flight during the barrier
  fetch();
  if (!grid_barrier(d.bar, abort_flag, a.status)) {
    cp_async_wait_all();
    return;
  }
  // h, written by every CTA, into shared memory
  const int vec = a.m.nb * 8;
  for (int i = threadIdx.x; i < R * vec; i += kW4Threads) {
    const int r = i / vec, v = i - r * vec;
    cp_async_16(smem_u32(hs) + r * pitch + v * 16, a.act + (static_cast<size_t>(r) * vec + v) * 4,
                16);
  }
  cp_async_wait_all();
  __syncthreads();

  int slot = 0, buffer = 0;
  for (int tile = blockIdx.x; tile < a.m.tiles; tile += grid) {
    for (int item = sh.tl; item < nitems; item += p.tl) {
      const int rec0 = items[item].y, n = items[item].z - rec0;
      uint32_t b[KB][8];
      float fold[KB][2], acc[4];
      const uint32_t src = smem_u32(hs) + (rec0 + min(g, n - 1)) * pitch + sh.kb0 * 128 + t * 4;
#pragma unroll
      for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          b[k][i] = g < n && k < sh.myb ? lds32(src + k * 128 + i * 16) : 0u;
      w4_fold<KB, MODE>(b, fold);
      cp_async_wait_group<1>();
      __syncwarp();  // every lane's copies of this tile have landed
      w4_tile<KB, MODE>(a, base + slot * p.slot_bytes, b, fold, acc);
      slot ^= 1;
      __syncwarp();  // and every lane has read them
      fetch();
      w4_meet(a, sh, acc, part, buffer);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int rec = 2 * t + u;
        if ((u & (p.ks - 1)) == sh.ks && rec < n) {
          dsum[rec0 + rec][g] = acc[u];
          dsum[rec0 + rec][g + 8] = acc[u + 2];
        }
      }
      buffer ^= kW4Warps * 128;
    }
    __syncthreads();
    // y = sum over the token's slots, in slot order, rounded once
    for (int i = threadIdx.x; i < d.T * 16; i += kW4Threads) {
      const int n = i >> 4, row = i & 15;
      float s = 0.0f;
      for (int j = 0; j < d.k; ++j)
        s = fmaf(rs.w[n * d.k + j], dsum[rs.pos[n * d.k + j]][row], s);
      d.y[static_cast<size_t>(n) * (a.m.tiles * 16) + tile * 16 + row] = __float2bfloat16_rn(s);
    }
    __syncthreads();
  }
  cp_async_wait_all();
}

// This group's share of the units (item, tile), split evenly over all groups of
// the grid, and a walk through it as w4_units takes it.
struct W4ItemWalk {
  const int4* items;
  int item, tile, hi_item, hi_tile;
  __device__ __forceinline__ W4ItemWalk(const W4Args& a, const int4* its, int nitems) : items(its) {
    const uint32_t tiles = a.m.tiles, total = nitems * tiles;
    const uint32_t parts = gridDim.x * a.p.tl;  // total * parts < 2^16 * 2^12
    const uint32_t part = blockIdx.x * a.p.tl + (threadIdx.x >> 5 >> a.p.ks_shift);
    const uint32_t lo = total * part / parts, hi = total * (part + 1) / parts;
    item = lo / tiles;
    tile = lo - item * tiles;
    hi_item = hi / tiles;
    hi_tile = hi - hi_item * tiles;
  }
  __device__ __forceinline__ int expert() const { return items[item].x; }
  __device__ __forceinline__ int first() const { return items[item].y; }
  __device__ __forceinline__ int count() const { return items[item].z - items[item].y; }
  __device__ __forceinline__ int run(const W4Args& a) {
    while (tile >= a.m.tiles) {
      tile -= a.m.tiles;
      ++item;
    }
    if (item > hi_item) return 0;
    return max((item == hi_item ? hi_tile : a.m.tiles) - tile, 0);
  }
};

template <int KB_UP, int KB_DOWN, int MODE>
__global__ void __launch_bounds__(kW4Threads, 1) w4_layer(const W4LayerArgs d) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ RouteSmem rs;
  __shared__ int4 items[kFusedMaxRecs];  // {expert, first record, last + 1, 0}
  __shared__ int nitems, abort_word;
  volatile int* abort_flag = &abort_word;
  if (threadIdx.x == 0) abort_word = 0;
  pdl_wait();
  pdl_trigger();
  topk_and_sort(d.logits, d.T, d.E, d.k, d.norm_topk_prob, rs);
  if (threadIdx.x < 32) {
    // Items: every expert's records by eights (32 lanes, two tiles each; 64 at most).
    const int lane = threadIdx.x;
    int chunks[2], at = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = 2 * lane + i;
      chunks[i] = e < rs.nt ? (rs.tiles[e].z - rs.tiles[e].y + kW4Recs - 1) / kW4Recs : 0;
    }
    at = chunks[0] + chunks[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += y;
    }
    if (lane == 31) nitems = at;
    at -= chunks[0] + chunks[1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      for (int c = 0; c < chunks[i]; ++c, ++at) {
        const int4 t = rs.tiles[2 * lane + i];
        const int first = t.y + c * kW4Recs;
        items[at] = make_int4(t.x, first, min(t.z, first + kW4Recs), 0);
      }
    }
  }
  __syncthreads();

  W4Args a = d.up;
  a.index = rs.perm;
  a.index_div = d.k;
  w4_units<true, KB_UP, MODE>(a, smem_raw + kW4PartBytes, reinterpret_cast<float*>(smem_raw),
                              W4ItemWalk(a, items, nitems));
  __syncthreads();  // every warp has left its slots
  w4_down<KB_DOWN, MODE>(d, rs, smem_raw, items, nitems, abort_flag);
}

template <int KB_UP, int KB_DOWN, int MODE>
int layer_launch(W4LayerArgs& d, cudaStream_t stream) {
  d.up.p = w4_plan(d.up.m, KB_UP);
  d.down.p = w4_plan(d.down.m, KB_DOWN);
  const int up = kW4PartBytes + kW4Warps * w4_slots<KB_UP, MODE>() * d.up.p.slot_bytes;
  const int down = kW4PartBytes + kW4Warps * kLayerSlots * d.down.p.slot_bytes +
                   kDsumBytes + d.T * d.k * h_pitch(64 * d.down.m.nb);
  const int sh = std::max(up, down);
  if (sh > kLayerSmemBytes) return kRcUnsupported;
  auto* kernel = w4_layer<KB_UP, KB_DOWN, MODE>;
  static std::atomic<uint64_t> attr{0};
  if (!allow_smem(kernel, kLayerSmemBytes, attr)) return kRcCudaError;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(device_sm_count());
  cfg.blockDim = dim3(kW4Threads);
  cfg.dynamicSmemBytes = sh;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeCooperative;  // every CTA resident: the grid barrier needs it
  attrs[0].val.cooperative = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = 2;
  return note_cuda_error(cudaLaunchKernelEx(&cfg, kernel, d)) == cudaSuccess ? kRcOk : kRcCudaError;
}

template <int MODE>
int layer_dispatch(W4LayerArgs& d, cudaStream_t stream) {
  const bool up8 = w4_best_kb(d.up.m.nb, {6, 8}) == 8, down8 = w4_best_kb(d.down.m.nb, {6, 8}) == 8;
  if (up8)
    return down8 ? layer_launch<8, 8, MODE>(d, stream) : layer_launch<8, 6, MODE>(d, stream);
  return down8 ? layer_launch<6, 8, MODE>(d, stream) : layer_launch<6, 6, MODE>(d, stream);
}

}  // namespace

bool w4_decode_ok(const W4Bank& b, int T, int k) {
  const W4Matrix m = w4_matrix(b, true);
  const int kb = w4_best_kb(m.nb, {6, 8});
  if (T < 1 || T > kLayerMaxT || T * k > kFusedMaxRecs || kb == 0) return false;
  const int down = kW4PartBytes + kW4Warps * kLayerSlots * w4_plan(m, kb).slot_bytes +
                   kDsumBytes + T * k * h_pitch(b.I);
  return router_small_ok(T, b.H, b.E, k) && w4_best_kb(b.H / 64, {6, 8}) > 0 &&
         down <= kLayerSmemBytes;
}

size_t w4_decode_scratch_bytes(const W4Bank& b, int T) {
  return static_cast<size_t>(T) * b.E * sizeof(float) + 256;
}

int launch_w4_decode(const W4Bank& b, const void* x, const void* wr, const float* bias, int T,
                     int k, int norm_topk_prob, void* scratch, void* h, void* y, int* status,
                     cudaStream_t stream) {
  if (!w4_decode_ok(b, T, k)) return kRcUnsupported;
  if (!aligned16(x) || !aligned16(wr) || !aligned16(h) || !aligned16(scratch))
    return kRcBadArgument;
  W4LayerArgs d{};
  d.x = static_cast<const uint4*>(x);
  d.T = T;
  d.k = k;
  d.E = b.E;
  d.norm_topk_prob = norm_topk_prob;
  d.bar = static_cast<unsigned int*>(scratch);
  float* logits = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + 256);
  d.logits = logits;
  d.y = static_cast<__nv_bfloat16*>(y);
  d.up.m = w4_matrix(b, false);
  d.up.act = static_cast<const uint32_t*>(x);
  d.up.act_rows = T;
  d.up.M = T * k;
  d.up.E = b.E;
  d.up.out = static_cast<__nv_bfloat16*>(h);
  d.up.out_ld = b.I;
  d.up.out_rows = T * k;
  d.up.status = status;
  d.down.m = w4_matrix(b, true);
  d.down.act = static_cast<const uint32_t*>(h);
  d.down.status = status;
  if (note_cuda_error(launch_pdl(w4_logits, dim3(T * b.E), dim3(32), 0, stream,
                                 static_cast<const uint4*>(x), static_cast<const uint4*>(wr), bias,
                                 b.H / 8, b.E, logits, d.bar)) != cudaSuccess)
    return kRcCudaError;
  if (d.up.m.rec == 8 || d.up.m.gshift == 0) return layer_dispatch<kW4Half>(d, stream);
  return d.up.m.gshift == 1 ? layer_dispatch<kW4Block>(d, stream)
                            : layer_dispatch<kW4TwoBlocks>(d, stream);
}

}  // namespace moe
