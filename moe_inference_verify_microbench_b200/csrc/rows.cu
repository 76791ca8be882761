// Row movement kernels: the permutation gather and the top-k combine.
//
// gather_rows   dst[p] = src[idx[p] / idx_div], p < min(R, *count)  (C5:135-137 gather
//               x_flat[token_ids_rep[perm]]; C7:167, C7:227 re-sort of received rows)
// combine_rows  y[n] = sum_j  w_j * rows[src_j]               (C5:158-160
//               weight scale + index_add_, C7:259-261, C8:221-224)
//               with src_j = slot_src ? slot_src[n*k+j] : n*k+j and w_j = slot_w ?
//               slot_w[n*k+j] : 1; a slot is skipped when src_j < 0 or when its
//               expert id (ids[n*k+j]) lies outside [e_begin, e_end).
//
// Both are HBM-bound copies with 16-byte vector accesses; the combine sums the
// k contributions in fp32 in slot order (deterministic, unlike the atomic
// index_add_ of the reference on CUDA).
#include <algorithm>
#include <atomic>

#include "internal.h"

namespace moe {

constexpr int kRowsThreads = 256;
constexpr int kRowsWarps = kRowsThreads / 32;

__global__ void __launch_bounds__(kRowsThreads) gather_rows(const uint4* __restrict__ src,
                                                            int src_rows,
                                                            const int* __restrict__ idx, int R,
                                                            const int* __restrict__ count,
                                                            int idx_div, int vec_per_row,
                                                            uint4* __restrict__ dst, int* status) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = count != nullptr ? min(R, *count) : R;
  for (int p = blockIdx.x * kRowsWarps + warp; p < rows; p += gridDim.x * kRowsWarps) {
    const int s = idx[p] / idx_div;
    if (s < 0 || s >= src_rows) {
      if (lane == 0) record_status(status, kErrBadRow);
      continue;
    }
    const uint4* a = src + static_cast<size_t>(s) * vec_per_row;
    uint4* b = dst + static_cast<size_t>(p) * vec_per_row;
    // Eight loads in flight per lane before the stores; the gathered rows are
    // written with the streaming hint so the source rows (each read k times)
    // keep their place in L2.
    for (int v0 = 0; v0 < vec_per_row; v0 += 8 * 32) {
      uint4 buf[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int v = v0 + u * 32 + lane;
        if (v < vec_per_row) buf[u] = __ldg(a + v);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int v = v0 + u * 32 + lane;
        if (v < vec_per_row) __stcs(b + v, buf[u]);
      }
    }
  }
}

constexpr int kCombineMaxK = 8;  // the router selects at most 8 experts

// One thread per (token, 16-byte column vector): the k source rows' vectors are
// loaded independently (no dependent chain of round trips), summed in fp32 in
// slot order, and stored once.
__global__ void __launch_bounds__(kRowsThreads) combine_rows(
    const uint4* __restrict__ rows, int n_rows, const int* __restrict__ slot_src,
    const float* __restrict__ slot_w, const int* __restrict__ ids, int e_begin, int e_end, int T,
    int k, int vec_per_row, uint4* __restrict__ y, int* status) {
  pdl_wait();
  pdl_trigger();
  const long long total = static_cast<long long>(T) * vec_per_row;
  for (long long g = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; g < total;
       g += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int n = static_cast<int>(g / vec_per_row);
    const int v = static_cast<int>(g - static_cast<long long>(n) * vec_per_row);
    uint4 val[kCombineMaxK];
    float wt[kCombineMaxK];
#pragma unroll
    for (int j = 0; j < kCombineMaxK; ++j) {
      wt[j] = 0.0f;
      val[j] = make_uint4(0u, 0u, 0u, 0u);
      if (j < k) {
        const int s = n * k + j;
        int src = slot_src != nullptr ? __ldg(slot_src + s) : s;
        if (ids != nullptr) {
          const int e = __ldg(ids + s);
          if (e < e_begin || e >= e_end) src = -1;
        }
        if (src >= n_rows) {
          record_status(status, kErrBadRow);
          src = -1;
        }
        if (src >= 0) {
          wt[j] = slot_w != nullptr ? __ldg(slot_w + s) : 1.0f;
          val[j] = __ldg(rows + static_cast<size_t>(src) * vec_per_row + v);
        }
      }
    }
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kCombineMaxK; ++j)
      if (j < k) acc_bf16x8(acc, val[j], wt[j]);
    uint4 o;
    o.x = pack_bf16x2(acc[0], acc[1]);
    o.y = pack_bf16x2(acc[2], acc[3]);
    o.z = pack_bf16x2(acc[4], acc[5]);
    o.w = pack_bf16x2(acc[6], acc[7]);
    y[g] = o;
  }
}

// The same over fp32 rows, row s of slot s, four columns a thread: the experts of a few
// tokens (a few MB at most, which stay in L2) need not be rounded before they are summed.
__global__ void __launch_bounds__(kRowsThreads) combine_rows_f32(
    const float4* __restrict__ rows, const int* __restrict__ ids, int e_begin, int e_end, int T,
    int k, int vec_per_row, uint2* __restrict__ y) {
  pdl_wait();
  pdl_trigger();
  const int total = T * vec_per_row;
  for (int g = blockIdx.x * blockDim.x + threadIdx.x; g < total; g += gridDim.x * blockDim.x) {
    const int n = g / vec_per_row, v = g - n * vec_per_row;
    float4 val[kCombineMaxK];
#pragma unroll
    for (int j = 0; j < kCombineMaxK; ++j) {
      val[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j < k) {
        const int s = n * k + j, e = __ldg(ids + s);
        if (e >= e_begin && e < e_end) val[j] = __ldg(rows + static_cast<size_t>(s) * vec_per_row + v);
      }
    }
    float4 acc = val[0];
#pragma unroll
    for (int j = 1; j < kCombineMaxK; ++j) {
      acc.x += val[j].x;
      acc.y += val[j].y;
      acc.z += val[j].z;
      acc.w += val[j].w;
    }
    y[g] = make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
  }
}

// Large batches: one warp per token, each lane sums 16-byte vectors of the k
// rows.  All loads of COLS column vectors are issued before any is used
// (KMAX x COLS = 16 loads in flight per lane), so a small k (the per-owner
// partial rows of the expert-parallel combine) still keeps 16 in flight.
template <int KMAX, int COLS>
__global__ void __launch_bounds__(kRowsThreads) combine_rows_warp(
    const uint4* __restrict__ rows, int n_rows, const int* __restrict__ slot_src,
    const float* __restrict__ slot_w, const int* __restrict__ ids, int e_begin, int e_end, int T,
    int k, int vec_per_row, uint4* __restrict__ y, int* status) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int n = blockIdx.x * kRowsWarps + warp; n < T; n += gridDim.x * kRowsWarps) {
    int src = -1;
    float w = 0.0f;
    if (lane < k) {
      const int s = n * k + lane;
      src = slot_src != nullptr ? slot_src[s] : s;
      w = slot_w != nullptr ? slot_w[s] : 1.0f;
      if (ids != nullptr) {
        const int e = ids[s];
        if (e < e_begin || e >= e_end) src = -1;
      }
      if (src >= n_rows) {
        record_status(status, kErrBadRow);
        src = -1;
      }
    }
    // The k source rows and weights, shuffled out once per token.
    int sj[KMAX];
    float wj[KMAX];
#pragma unroll
    for (int j = 0; j < KMAX; ++j) {
      sj[j] = __shfl_sync(0xffffffffu, src, j);
      wj[j] = __shfl_sync(0xffffffffu, w, j);
      if (j >= k) sj[j] = -1;
    }
    for (int v0 = 0; v0 < vec_per_row; v0 += 32 * COLS) {
      uint4 val[COLS][KMAX];
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const int v = v0 + 32 * c + lane;
#pragma unroll
        for (int j = 0; j < KMAX; ++j) {
          val[c][j] = make_uint4(0, 0, 0, 0);
          if (sj[j] >= 0 && v < vec_per_row)
            val[c][j] = __ldg(rows + static_cast<size_t>(sj[j]) * vec_per_row + v);
        }
      }
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const int v = v0 + 32 * c + lane;
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KMAX; ++j)  // slot order, as the reference sums
          if (sj[j] >= 0) acc_bf16x8(acc, val[c][j], wj[j]);
        if (v < vec_per_row) {
          uint4 o;
          o.x = pack_bf16x2(acc[0], acc[1]);
          o.y = pack_bf16x2(acc[2], acc[3]);
          o.z = pack_bf16x2(acc[4], acc[5]);
          o.w = pack_bf16x2(acc[6], acc[7]);
          y[static_cast<size_t>(n) * vec_per_row + v] = o;
        }
      }
    }
  }
}

// y = bf16(src), eight elements per thread (two 16-byte loads, one 16-byte
// store): the final rounding of the atomic combine's fp32 accumulation rows.
__global__ void __launch_bounds__(kRowsThreads) cast_f32_bf16(const float4* __restrict__ src,
                                                              long long n8, uint4* __restrict__ y) {
  pdl_wait();
  pdl_trigger();
  for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < n8;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const float4 a = __ldcs(src + 2 * i), b = __ldcs(src + 2 * i + 1);
    y[i] = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y),
                      pack_bf16x2(b.z, b.w));
  }
}

// Pre-norm decoder block glue (the residual add and RMSNorm around the MoE of
// C8/python/solution.py:235-325, RMSNorm as the suite's harness defines it):
//   h = delta ? bf16(x + delta) : x
//   y = bf16((float(h) * rsqrt(mean_j float(h_j)^2 + eps)) * w)
// one warp per row, fp32 throughout, the row's sum of squares reduced across
// the warp; the second pass re-reads the row (L1/L2 hits).
__global__ void __launch_bounds__(kRowsThreads) add_rmsnorm_rows(
    const uint4* __restrict__ x, const uint4* __restrict__ delta, const float* __restrict__ w,
    int T, int vec, float eps, uint4* __restrict__ h_out, uint4* __restrict__ y) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float inv_h = 1.0f / static_cast<float>(vec * 8);
  for (int n = blockIdx.x * kRowsWarps + warp; n < T; n += gridDim.x * kRowsWarps) {
    const uint4* xr = x + static_cast<size_t>(n) * vec;
    const uint4* dr = delta != nullptr ? delta + static_cast<size_t>(n) * vec : nullptr;
    float ss = 0.0f;
    for (int v = lane; v < vec; v += 32) {
      uint4 a = __ldg(xr + v);
      if (dr != nullptr) {
        const uint4 b = __ldg(dr + v);
        const __nv_bfloat162* a2 = reinterpret_cast<const __nv_bfloat162*>(&a);
        const __nv_bfloat162* b2 = reinterpret_cast<const __nv_bfloat162*>(&b);
        uint32_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 fa = __bfloat1622float2(a2[q]), fb = __bfloat1622float2(b2[q]);
          o[q] = pack_bf16x2(fa.x + fb.x, fa.y + fb.y);
        }
        a = make_uint4(o[0], o[1], o[2], o[3]);
        h_out[static_cast<size_t>(n) * vec + v] = a;
      }
      const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 f = __bfloat1622float2(h2[q]);
        ss = fmaf(f.x, f.x, ss);
        ss = fmaf(f.y, f.y, ss);
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * inv_h + eps);
    // Each lane re-reads only the h_out vectors it stored itself.
    const uint4* hr = dr != nullptr ? h_out + static_cast<size_t>(n) * vec : xr;
    for (int v = lane; v < vec; v += 32) {
      const uint4 a = dr != nullptr ? hr[v] : __ldg(hr + v);
      const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&a);
      const float4 w0 = __ldg(reinterpret_cast<const float4*>(w) + 2 * v);
      const float4 w1 = __ldg(reinterpret_cast<const float4*>(w) + 2 * v + 1);
      const float wv[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
      uint32_t o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 f = __bfloat1622float2(h2[q]);
        o[q] = pack_bf16x2((f.x * r) * wv[2 * q], (f.y * r) * wv[2 * q + 1]);
      }
      y[static_cast<size_t>(n) * vec + v] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// The norm after a block, its gate and residual scale, and the norm before the
// next block, in one pass over the rows:
//   n = delta * rsqrt(mean(delta^2) + eps) * post
//   h = x + scale * act(gate) * n
//   y = h * rsqrt(mean(h^2) + eps) * pre
// HBM bounds it: 4 H bytes read and 4 H written per row (and the gate).  One
// CTA per row keeps x, delta and then h in registers (VPT 16-byte vectors per
// thread), so nothing is read twice; both sums of squares and h are fp32, and y
// is the norm of the unrounded h.
// The sigmoid and tanh by one exponential each: tanh x = sign(x) (1 - e) / (1 + e),
// e = exp(-2 |x|), whose difference loses bits near zero, so below 2^-6 it is
// x - x^3 / 3 (the next term is 2 x^4 / 15 < 2^-26 of it).
template <int ACT>
__device__ __forceinline__ float gate_act(float g) {
  if (ACT == 1) return __fdividef(1.0f, 1.0f + __expf(-g));
  if (ACT == 2) {
    const float a = fabsf(g);
    const float e = __expf(-2.0f * a);
    const float t = copysignf(__fdividef(1.0f - e, 1.0f + e), g);
    return a < 0.015625f ? fmaf(g * g * g, -1.0f / 3.0f, g) : t;
  }
  return g;
}

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 p = __bfloat1622float2(h[q]);
    f[2 * q] = p.x;
    f[2 * q + 1] = p.y;
  }
}

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
  f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// Sum over the CTA; every thread gets it.  `sh` holds one float per warp.
__device__ __forceinline__ float cta_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = static_cast<int>(threadIdx.x & 31) < nw ? sh[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

constexpr int kBlockNormMaxH = 4 * 8 * 1024;

// Read once: past L1, and coherent, because h may be written over x and y over delta
// (a .nc load may only read what nothing writes while the kernel runs).
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

template <int VPT, int ACT, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS) block_norm_rows(const BlockNormArgs a) {
  __shared__ float sh[2][32];
  pdl_wait();
  pdl_trigger();
  const int vec = a.H / 8;
  const size_t n = blockIdx.x;
  const uint4* xr = static_cast<const uint4*>(a.x) + n * vec;
  const uint4* dr = static_cast<const uint4*>(a.delta) + n * vec;
  const bool gated = a.gate != nullptr && a.gate_col != 0, gate_bf16 = gated && !a.gate_f32;
  const __nv_bfloat16* gr = static_cast<const __nv_bfloat16*>(a.gate) + n * a.gate_row;
  uint4 xv[VPT], dv[VPT], gv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    xv[i] = dv[i] = gv[i] = make_uint4(0, 0, 0, 0);
    if (v < vec) {
      dv[i] = load_once(dr + v);
      xv[i] = load_once(xr + v);
      if (gate_bf16) gv[i] = load_once(reinterpret_cast<const uint4*>(gr) + v);
    }
  }
  float token_gate = 1.0f;  // one gate for the row
  if (a.gate != nullptr && a.gate_col == 0) {
    const float g = a.gate_f32 ? static_cast<const float*>(a.gate)[n * a.gate_row]
                               : __bfloat162float(gr[0]);
    token_gate = gate_act<ACT>(g);
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float d[8];
    unpack8(dv[i], d);
#pragma unroll
    for (int q = 0; q < 8; ++q) ss = fmaf(d[q], d[q], ss);
  }
  const float inv_h = 1.0f / static_cast<float>(a.H);
  const float r1 = rsqrtf(cta_sum(ss, sh[0]) * inv_h + a.eps) * a.scale;
  float h[VPT][8];
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
#pragma unroll
    for (int q = 0; q < 8; ++q) h[i][q] = 0.0f;
    if (v < vec) {
      float d[8], w[8], gt[8];
      unpack8(xv[i], h[i]);
      unpack8(dv[i], d);
      load8(a.post + 8 * v, w);
#pragma unroll
      for (int q = 0; q < 8; ++q) gt[q] = token_gate;
      if (gated) {
        if (gate_bf16) unpack8(gv[i], gt);
        else load8(static_cast<const float*>(a.gate) + n * a.gate_row + 8 * v, gt);
#pragma unroll
        for (int q = 0; q < 8; ++q) gt[q] = gate_act<ACT>(gt[q]);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        h[i][q] = fmaf(d[q] * r1 * w[q], gt[q], h[i][q]);
        ss = fmaf(h[i][q], h[i][q], ss);
      }
      static_cast<uint4*>(a.h)[n * vec + v] =
          make_uint4(pack_bf16x2(h[i][0], h[i][1]), pack_bf16x2(h[i][2], h[i][3]),
                     pack_bf16x2(h[i][4], h[i][5]), pack_bf16x2(h[i][6], h[i][7]));
    }
  }
  const float r2 = rsqrtf(cta_sum(ss, sh[1]) * inv_h + a.eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < vec) {
      float w[8];
      load8(a.pre + 8 * v, w);
      uint32_t o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        o[q] = pack_bf16x2(h[i][2 * q] * r2 * w[2 * q], h[i][2 * q + 1] * r2 * w[2 * q + 1]);
      static_cast<uint4*>(a.y)[n * vec + v] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// The same for many rows: persistent CTAs whose rows arrive through a ring of
// shared-memory stages by bulk copies (x, delta and, where there is one for every
// element, the gate), so that HBM reads never wait for a reduction.  A thread
// keeps its columns' weights in registers for all rows; a gate for each channel is
// multiplied into them once.
constexpr int kNormThreads = 256;
// CTAs per SM: a row is a chain of two reductions, so short rows want more of them.
template <int VPT>
constexpr int norm_ctas() {
  return VPT == 1 ? 4 : 2;
}
template <int VPT>
constexpr int norm_ring_bytes() {
  return (VPT == 1 ? 50 : 100) * 1024;
}
constexpr int kNormMaxStages = 8;

// Whether a stage's copies have landed, within the limit of every wait.
__device__ __forceinline__ bool norm_rows_wait(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > kWaitLimitNs) return false;
  return true;
}

template <int VPT, int ACT>
__global__ void __launch_bounds__(kNormThreads, norm_ctas<VPT>())
    block_norm_stream(const BlockNormArgs a,
                                                                     int stages) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float sh[2][8];
  __shared__ __align__(8) uint64_t full[kNormMaxStages];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vec = a.H / 8;
  const uint32_t row_bytes = static_cast<uint32_t>(a.H) * 2;
  const bool elem = a.gate != nullptr && a.gate_col != 0 && a.gate_row != 0;
  const uint32_t gate_bytes = elem ? (a.gate_f32 ? 2 * row_bytes : row_bytes) : 0u;
  const uint32_t stage_bytes = 2 * row_bytes + gate_bytes;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  auto fetch = [&](int row, int s) {  // one thread
    uint8_t* dst = ring + s * stage_bytes;
    const size_t o = static_cast<size_t>(row);
    mbar_arrive_expect_tx(&full[s], stage_bytes);
    bulk_load(dst, static_cast<const uint8_t*>(a.x) + o * row_bytes, row_bytes, &full[s]);
    bulk_load(dst + row_bytes, static_cast<const uint8_t*>(a.delta) + o * row_bytes, row_bytes,
              &full[s]);
    if (elem)
      bulk_load(dst + 2 * row_bytes, static_cast<const uint8_t*>(a.gate) + o * gate_bytes,
                gate_bytes, &full[s]);
  };
  const int grid = gridDim.x;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      const long long row = blockIdx.x + static_cast<long long>(s) * grid;
      if (row < a.T) fetch(static_cast<int>(row), s);
    }
  }
  float post[VPT][8], pre[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * kNormThreads;
    if (v < vec) {
      load8(a.post + 8 * v, post[i]);
      load8(a.pre + 8 * v, pre[i]);
      float g[8];
      if (a.gate != nullptr && a.gate_col != 0 && !elem) {
        if (a.gate_f32) load8(static_cast<const float*>(a.gate) + 8 * v, g);
        else unpack8(__ldg(static_cast<const uint4*>(a.gate) + v), g);
#pragma unroll
        for (int q = 0; q < 8; ++q) post[i][q] *= gate_act<ACT>(g[q]);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) post[i][q] *= a.scale;
    }
  }
  const float inv_h = 1.0f / static_cast<float>(a.H);
  int s = 0;
  uint32_t ph = 0;
  long long refill = -1;  // row to fetch into the stage before s, once every thread left it
  for (long long row = blockIdx.x; row < a.T; row += grid) {
    float token_gate = 1.0f;
    if (a.gate != nullptr && a.gate_col == 0)
      token_gate = gate_act<ACT>(
          a.gate_f32 ? static_cast<const float*>(a.gate)[row]
                     : __bfloat162float(static_cast<const __nv_bfloat16*>(a.gate)[row]));
    const bool late = !norm_rows_wait(&full[s], ph);
    const uint4* sx = reinterpret_cast<const uint4*>(ring + s * stage_bytes);
    const uint4* sd = sx + vec;
    float h[VPT][8], d[VPT][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * kNormThreads;
      if (v < vec) {
        unpack8(sd[v], d[i]);
#pragma unroll
        for (int q = 0; q < 8; ++q) ss = fmaf(d[i][q], d[i][q], ss);
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) sh[0][warp] = ss;
    // also: every thread has left the previous row's stage
    if (__syncthreads_or(late)) {
      // Nothing more is stored or asked for; what is on its way lands before the CTA
      // exits: the stages from s on, without the one before s, which waits for its refill.
      if (tid == 0) {
        record_status(a.status, kErrTimeoutRows);
        for (int j = 0; j < (row == blockIdx.x ? stages : stages - 1); ++j) {
          if (row + static_cast<long long>(j) * grid >= a.T) break;
          norm_rows_wait(&full[(s + j) % stages], s + j < stages ? ph : ph ^ 1u);
        }
      }
      return;
    }
    if (tid == 0 && refill >= 0) {
      fence_proxy_async_smem();
      fetch(static_cast<int>(refill), s == 0 ? stages - 1 : s - 1);
    }
    ss = 0.0f;
#pragma unroll
    for (int w = 0; w < kNormThreads / 32; ++w) ss += sh[0][w];
    const float r1 = rsqrtf(ss * inv_h + a.eps) * token_gate;
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * kNormThreads;
      if (v < vec) {
        unpack8(sx[v], h[i]);
        float g[8];
        if (elem) {
          const uint8_t* sg = reinterpret_cast<const uint8_t*>(sd + vec);
          if (a.gate_f32) {
            const float4 g0 = reinterpret_cast<const float4*>(sg)[2 * v];
            const float4 g1 = reinterpret_cast<const float4*>(sg)[2 * v + 1];
            g[0] = g0.x, g[1] = g0.y, g[2] = g0.z, g[3] = g0.w;
            g[4] = g1.x, g[5] = g1.y, g[6] = g1.z, g[7] = g1.w;
          } else {
            unpack8(reinterpret_cast<const uint4*>(sg)[v], g);
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) d[i][q] *= gate_act<ACT>(g[q]);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          h[i][q] = fmaf(d[i][q] * r1, post[i][q], h[i][q]);
          ss = fmaf(h[i][q], h[i][q], ss);
        }
        static_cast<uint4*>(a.h)[static_cast<size_t>(row) * vec + v] =
            make_uint4(pack_bf16x2(h[i][0], h[i][1]), pack_bf16x2(h[i][2], h[i][3]),
                       pack_bf16x2(h[i][4], h[i][5]), pack_bf16x2(h[i][6], h[i][7]));
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) sh[1][warp] = ss;
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int w = 0; w < kNormThreads / 32; ++w) ss += sh[1][w];
    const float r2 = rsqrtf(ss * inv_h + a.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * kNormThreads;
      if (v < vec) {
        uint32_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          o[q] = pack_bf16x2(h[i][2 * q] * r2 * pre[i][2 * q],
                             h[i][2 * q + 1] * r2 * pre[i][2 * q + 1]);
        static_cast<uint4*>(a.y)[static_cast<size_t>(row) * vec + v] =
            make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    refill = row + static_cast<long long>(stages) * grid;
    if (refill >= a.T) refill = -1;
    if (++s == stages) {
      s = 0;
      ph ^= 1u;
    }
  }
}

static int rows_grid(long long rows) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long want = (rows + kRowsWarps - 1) / kRowsWarps;
  const long long cap = static_cast<long long>(sms) * 8;
  return static_cast<int>(want < cap ? (want > 0 ? want : 1) : cap);
}

int launch_gather_rows(const void* src, int src_rows, const int* idx, int R, const int* count,
                       int idx_div, int H, void* dst, int* status, cudaStream_t stream) {
  if (R < 0 || H <= 0 || idx_div <= 0 || (H % 8) != 0) return kRcBadArgument;
  if (R == 0) return kRcOk;
  const cudaError_t e = launch_pdl(gather_rows, dim3(rows_grid(R)), dim3(kRowsThreads), 0, stream,
                                   static_cast<const uint4*>(src), src_rows, idx, R, count,
                                   idx_div, H / 8, static_cast<uint4*>(dst), status);
  return e == cudaSuccess ? kRcOk : kRcCudaError;
}

int launch_combine(const void* rows, int n_rows, const int* slot_src, const float* slot_w,
                   const int* ids, int e_begin, int e_end, int T, int k, int H, void* y,
                   int* status, cudaStream_t stream) {
  if (T < 0 || k <= 0 || k > kCombineMaxK || H <= 0 || (H % 8) != 0) return kRcBadArgument;
  if (T == 0) return kRcOk;
  if (T >= 1024) {
    auto kern = k > 4 ? combine_rows_warp<8, 2> : k > 2 ? combine_rows_warp<4, 4>
                                                        : combine_rows_warp<2, 8>;
    const cudaError_t e = launch_pdl(kern, dim3(rows_grid(T)), dim3(kRowsThreads), 0, stream,
                                     static_cast<const uint4*>(rows), n_rows, slot_src, slot_w,
                                     ids, e_begin, e_end, T, k, H / 8, static_cast<uint4*>(y),
                                     status);
    return e == cudaSuccess ? kRcOk : kRcCudaError;
  }
  const long long threads = static_cast<long long>(T) * (H / 8);
  const long long blocks = (threads + kRowsThreads - 1) / kRowsThreads;
  const int grid = static_cast<int>(blocks < 148LL * 16 ? blocks : 148LL * 16);
  const cudaError_t e = launch_pdl(combine_rows, dim3(grid), dim3(kRowsThreads), 0, stream,
                                   static_cast<const uint4*>(rows), n_rows, slot_src, slot_w, ids,
                                   e_begin, e_end, T, k, H / 8, static_cast<uint4*>(y), status);
  return e == cudaSuccess ? kRcOk : kRcCudaError;
}

int launch_combine_f32(const float* rows, const int* ids, int e_begin, int e_end, int T, int k,
                       int H, void* y, cudaStream_t stream) {
  if (T < 0 || k <= 0 || k > kCombineMaxK || H <= 0 || (H % 4) != 0 ||
      static_cast<long long>(T) * H > 0x7fffffffLL)
    return kRcBadArgument;
  if (T == 0) return kRcOk;
  const int blocks = (T * (H / 4) + kRowsThreads - 1) / kRowsThreads;
  const cudaError_t e =
      launch_pdl(combine_rows_f32, dim3(blocks), dim3(kRowsThreads), 0, stream,
                 reinterpret_cast<const float4*>(rows), ids, e_begin, e_end, T, k, H / 4,
                 static_cast<uint2*>(y));
  return e == cudaSuccess ? kRcOk : kRcCudaError;
}

int launch_add_rmsnorm(const void* x, const void* delta, const float* w, int T, int H, float eps,
                       void* h_out, void* y, cudaStream_t stream) {
  if (T < 0 || H <= 0 || (H % 8) != 0 || !(eps >= 0.0f) ||
      (T > 0 && (x == nullptr || w == nullptr || y == nullptr ||
                 (delta != nullptr && h_out == nullptr))))
    return kRcBadArgument;
  for (const void* p : {x, delta, static_cast<const void*>(w), static_cast<const void*>(h_out),
                        static_cast<const void*>(y)})
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return kRcBadArgument;
  if (T == 0) return kRcOk;
  const cudaError_t e = launch_pdl(add_rmsnorm_rows, dim3(rows_grid(T)), dim3(kRowsThreads), 0,
                                   stream, static_cast<const uint4*>(x),
                                   static_cast<const uint4*>(delta), w, T, H / 8, eps,
                                   static_cast<uint4*>(h_out), static_cast<uint4*>(y));
  return e == cudaSuccess ? kRcOk : kRcCudaError;
}

template <int VPT, int MAX_THREADS = 1024>
static cudaError_t block_norm_launch(const BlockNormArgs& a, cudaStream_t stream) {
  const int vec = a.H / 8;
  const int threads = ((vec + VPT - 1) / VPT + 31) / 32 * 32;
  auto kern = a.act == 1   ? block_norm_rows<VPT, 1, MAX_THREADS>
              : a.act == 2 ? block_norm_rows<VPT, 2, MAX_THREADS>
                           : block_norm_rows<VPT, 0, MAX_THREADS>;
  return launch_pdl(kern, dim3(a.T), dim3(threads), 0, stream, a);
}

template <int VPT>
static cudaError_t block_norm_stream_launch(const BlockNormArgs& a, int stage,
                                            cudaStream_t stream) {
  const int stages = std::min(kNormMaxStages, norm_ring_bytes<VPT>() / stage);
  auto kern = a.act == 1   ? block_norm_stream<VPT, 1>
              : a.act == 2 ? block_norm_stream<VPT, 2>
                           : block_norm_stream<VPT, 0>;
  static std::atomic<uint64_t> done{0};  // per device: the three kernels' limits are raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if ((done.load(std::memory_order_acquire) & bit) == 0) {
    for (auto* k : {block_norm_stream<VPT, 0>, block_norm_stream<VPT, 1>, block_norm_stream<VPT, 2>}) {
      e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               norm_ring_bytes<VPT>());
      if (e != cudaSuccess) return e;
    }
    done.fetch_or(bit, std::memory_order_acq_rel);
  }
  const int grid = std::min(a.T, norm_ctas<VPT>() * device_sm_count());
  return launch_pdl(kern, dim3(grid), dim3(kNormThreads), static_cast<size_t>(stage) * stages,
                    stream, a, stages);
}

int launch_block_norm(const BlockNormArgs& a, cudaStream_t stream) {
  if (a.T < 0 || a.H <= 0 || !(a.eps >= 0.0f) || a.act < 0 || a.act > 2 || a.gate_row < 0 ||
      (a.gate_col != 0 && a.gate_col != 1) ||
      (a.T > 0 && (a.x == nullptr || a.delta == nullptr || a.post == nullptr ||
                   a.pre == nullptr || a.h == nullptr || a.y == nullptr)))
    return kRcBadArgument;
  if (a.H % 8 != 0 || a.H > kBlockNormMaxH) return kRcUnsupported;
  for (const void* p : {a.x, a.delta, static_cast<const void*>(a.post),
                        static_cast<const void*>(a.pre), static_cast<const void*>(a.h),
                        static_cast<const void*>(a.y)})
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return kRcBadArgument;
  if (a.gate != nullptr && a.gate_col != 0 &&
      ((reinterpret_cast<uintptr_t>(a.gate) & 15u) != 0 || a.gate_row % 8 != 0))
    return kRcBadArgument;
  if (a.T == 0) return kRcOk;
  const int vec = a.H / 8;
  // Measured (ncu, L2 cold, B200).  Few rows are a latency: a thread for each vector
  // (333 x 2048: 4.6 us, two vectors a thread 5.6).  From about a thousand on
  // the rows in flight count: two vectors a thread (16384 x 2048: 49 us against 57),
  // four where a row is long (1200 x 8192: 24 us against 33).  Streaming rows through
  // shared memory wins once every CTA has many of them and its threads are busy
  // (16384 x 2048: 46 us; 9001 x 5120: 57 us against 72; 4096 x 2048: 16.6 against 15.1).
  const bool elem = a.gate != nullptr && a.gate_col != 0 && a.gate_row != 0;
  const int stage = a.H * (elem ? (a.gate_f32 ? 8 : 6) : 4);
  const int min_rows = vec <= kNormThreads ? 8192 : 2048;
  cudaError_t e;
  if (a.T >= min_rows && 2 * vec > kNormThreads && vec <= 4 * kNormThreads &&
      3 * stage <= norm_ring_bytes<2>())
    e = vec <= kNormThreads       ? block_norm_stream_launch<1>(a, stage, stream)
        : vec <= 2 * kNormThreads ? block_norm_stream_launch<2>(a, stage, stream)
        : vec <= 3 * kNormThreads ? block_norm_stream_launch<3>(a, stage, stream)
                                  : block_norm_stream_launch<4>(a, stage, stream);
  else if (a.T >= 1024 && vec > 512 && vec <= 1024)
    e = block_norm_launch<4, 256>(a, stream);
  else if (a.T >= 1024 && vec >= 128 && vec <= 512)
    e = block_norm_launch<2, 256>(a, stream);
  else
    e = vec <= 1024   ? block_norm_launch<1>(a, stream)
        : vec <= 2048 ? block_norm_launch<2>(a, stream)
                      : block_norm_launch<4>(a, stream);
  return note_cuda_error(e) == cudaSuccess ? kRcOk : kRcCudaError;
}

int launch_cast_f32_bf16(const float* src, long long n, void* y, cudaStream_t stream) {
  if (n < 0 || (n % 8) != 0 || (n > 0 && (src == nullptr || y == nullptr)) ||
      (reinterpret_cast<uintptr_t>(src) & 15u) != 0 || (reinterpret_cast<uintptr_t>(y) & 15u) != 0)
    return kRcBadArgument;
  if (n == 0) return kRcOk;
  const long long n8 = n / 8;
  const long long blocks = (n8 + kRowsThreads - 1) / kRowsThreads;
  const long long cap = static_cast<long long>(device_sm_count()) * 8;
  const int grid = static_cast<int>(blocks < cap ? blocks : cap);
  const cudaError_t e = launch_pdl(cast_f32_bf16, dim3(grid), dim3(kRowsThreads), 0, stream,
                                   reinterpret_cast<const float4*>(src), n8,
                                   static_cast<uint4*>(y));
  return e == cudaSuccess ? kRcOk : kRcCudaError;
}

}  // namespace moe
