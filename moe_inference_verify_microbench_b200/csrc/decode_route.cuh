// The routing pieces that the single-launch decode layers share (decode.cu,
// w4_decode.cu): dot products, the grid barrier, and the top-k and record sort that
// every CTA does for itself.
#pragma once

#include "grouped_gemm.cuh"

namespace moe {

constexpr int kFusedMaxRecs = 64;  // routing records of the single-launch layers (T*k)
constexpr int kRouterMaxVecPerLane = 16;  // H <= 32 * 16 * 8 = 4096

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Mixed-precision FMA: fma.rn.f32.bf16 multiplies two bf16 values exactly and
// adds them to an fp32 accumulator with one rounding, so weights and
// activations are used as stored, without conversion instructions.
__device__ __forceinline__ void fma_bf16x2(float& lo, float& hi, uint32_t w, uint32_t x) {
  asm("{\n\t.reg .b16 wl, wh, xl, xh;\n\t"
      "mov.b32 {wl, wh}, %2;\n\t"
      "mov.b32 {xl, xh}, %3;\n\t"
      "fma.rn.f32.bf16 %0, wl, xl, %0;\n\t"
      "fma.rn.f32.bf16 %1, wh, xh, %1;\n\t}"
      : "+f"(lo), "+f"(hi)
      : "r"(w), "r"(x));
}

// acc[0..3] += the 8-element dot product of w and x, over four dependency chains.
__device__ __forceinline__ void dot8_acc(const uint4& w, const uint4& x, float* acc) {
  fma_bf16x2(acc[0], acc[1], w.x, x.x);
  fma_bf16x2(acc[2], acc[3], w.y, x.y);
  fma_bf16x2(acc[0], acc[1], w.z, x.z);
  fma_bf16x2(acc[2], acc[3], w.w, x.w);
}

__device__ __forceinline__ float acc_sum(const float* acc) {
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

// All CTAs of the grid arrive on *ctr and wait until gridDim.x have arrived.
// False (and the CTA's abort flag raised) once the bounded wait gives up or
// the CTA has aborted before.
__device__ inline bool grid_barrier(unsigned int* ctr, volatile int* abort_flag, int* status) {
  __syncthreads();
  if (threadIdx.x == 0 && !*abort_flag) {
    __threadfence();
    atomicAdd(ctr, 1u);
    const unsigned long long t0 = globaltimer_ns();
    for (;;) {
      unsigned int v;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(ctr) : "memory");
      if (v >= gridDim.x) break;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        record_status(status, kErrTimeoutGrid);
        *abort_flag = 1;
        break;
      }
      __nanosleep(32);
    }
    __threadfence();
  }
  __syncthreads();
  return *abort_flag == 0;
}

struct RouteSmem {
  int ids[kFusedMaxRecs];
  int first[kFusedMaxRecs];    // 1: the record opens its expert's tile
  float w[kFusedMaxRecs];      // routing weight of slot n*k + j
  int perm[kFusedMaxRecs];     // slot of the p-th record in expert order
  int pos[kFusedMaxRecs];      // position of slot s in expert order
  int tile_of[kFusedMaxRecs];  // tile of slot s
  int4 tiles[kFusedMaxRecs];
  int nt;
};

// The top-k of every token from its logits [T][E] (each warp of the CTA takes
// tokens in turn) and the stable sort of the T * k records by expert, one tile per
// expert, into rs.  Every thread of the CTA calls it.
__device__ __forceinline__ void topk_and_sort(const float* logits, int T, int E, int k,
                                              int norm_topk_prob, RouteSmem& rs) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = T * k;
  for (int t = warp; t < T; t += static_cast<int>(blockDim.x >> 5)) {  // one warp per token
    const float* lg = logits + t * E;
    uint32_t top[kRouterMaxK];
#pragma unroll
    for (int i = 0; i < kRouterMaxK; ++i) top[i] = 0u;
    for (int c = lane; c < E; c += 32) topk_insert(top, topk_key(__ldcg(lg + c), c));
    uint32_t sel[kRouterMaxK];
#pragma unroll
    for (int i = 0; i < kRouterMaxK; ++i) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, top[0]);
      sel[i] = m;
      if (top[0] == m) {
#pragma unroll
        for (int j = 0; j + 1 < kRouterMaxK; ++j) top[j] = top[j + 1];
        top[kRouterMaxK - 1] = 0u;
      }
    }
    const float ref = topk_key_value(sel[0]);
    float den = 0.0f;
    if (norm_topk_prob) {
#pragma unroll
      for (int i = 0; i < kRouterMaxK; ++i)
        if (i < k) den += expf(topk_key_value(sel[i]) - ref);
    } else {
      for (int c = lane; c < E; c += 32) den += expf(__ldcg(lg + c) - ref);
      den = warp_sum(den);
    }
    const float inv = 1.0f / den;
#pragma unroll
    for (int i = 0; i < kRouterMaxK; ++i) {
      if (i < k && lane == i) {
        rs.ids[t * k + i] = topk_key_id(sel[i]);
        rs.w[t * k + i] = expf(topk_key_value(sel[i]) - ref) * inv;
      }
    }
  }
  __syncthreads();
  // Stable sort of the R <= kFusedMaxRecs records by expert, thread r =
  // slot r, over the ids in shared memory: a record's position counts the
  // records with a smaller id or the same id and a lower slot; one tile per
  // expert, ascending ids (the first record of an expert opens its tile).
  const int r = static_cast<int>(threadIdx.x);
  int my = 0x7fffffff, pos = 0, before = 0, same = 0;
  bool first = false;
  if (r < R) {
    my = rs.ids[r];
    first = true;
    for (int j = 0; j < R; ++j) {
      const int o = rs.ids[j];
      pos += (o < my || (o == my && j < r)) ? 1 : 0;
      before += o < my ? 1 : 0;
      same += o == my ? 1 : 0;
      if (o == my && j < r) first = false;
    }
    rs.first[r] = first ? 1 : 0;
  }
  __syncthreads();
  if (r < R) {
    int tile = 0, n_tiles = 0;
    for (int j = 0; j < R; ++j) {
      const bool f = rs.first[j] != 0;
      tile += (f && rs.ids[j] < my) ? 1 : 0;
      n_tiles += f ? 1 : 0;
    }
    rs.perm[pos] = r;
    rs.pos[r] = pos;
    rs.tile_of[r] = tile;
    if (first) rs.tiles[tile] = make_int4(my, before, before + same, 0);
    if (r == 0) rs.nt = n_tiles;
  }
  __syncthreads();
}

}  // namespace moe
