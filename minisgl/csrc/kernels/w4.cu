// Products with 4-bit weights and group scales: w[n, k] = (code - zero) * scale(row n, group of k).
//
// Packed weights (ops/w4.py lays them out once): tiles of 16 rows by 64 inputs, 512 bytes each, in the
// order of the tensor core's A fragments, so that a warp's 16-byte loads are one tile:
//   q [E][Nt][KB][32 lanes][4 words], lane = 4 g + t. Word 2h + j holds, for k = 64 kb + 32 h + 8 t + 4 j,
//     row g     codes k, k+1, k+2, k+3 in nibbles 0, 4, 2, 6
//     row g + 8 codes k, k+1, k+2, k+3 in nibbles 1, 5, 3, 7
//   s [E][Nt][KG][8][2] 16-bit scales of rows g and g + 8, z likewise in bytes (none: 8).
// Rows and inputs are padded to whole tiles with scales of zero. In a gated weight rows 0-7 of a tile
// are gate rows 8 i .. 8 i + 7 and rows 8-15 the up rows of the same outputs.
#include <cuda_fp16.h>

#include <algorithm>

#include "api.h"
#include "common.cuh"

using namespace msgl;

namespace {

struct W4Tensor {
  const uint4* q;
  const uint32_t* s;  // two 16-bit scales
  const uint16_t* z;  // two zero points, or null
  int tiles, kb, kg, group, n, k, fp16;
};

__device__ __forceinline__ float2 scale2(uint32_t v, int fp16) {
  if (fp16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  return make_float2(bf16_lo(v), bf16_hi(v));
}

// acc[m][0/1] += rows g and g + 8 of tile (e, nt) times x[m] over 64-input blocks kb0, kb0 + step, ...
template <int MT>
__device__ __forceinline__ void tile_dot(const W4Tensor& w, int64_t tile, const __nv_bfloat16* const (&x)[MT], int kb0,
                                         int step, float (&acc)[MT][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint4* q = w.q + tile * w.kb * 32 + lane;
  const uint32_t* s = w.s + tile * w.kg * 8 + g;
  const uint16_t* z = w.z == nullptr ? nullptr : w.z + tile * w.kg * 8 + g;
  for (int kb = kb0; kb < w.kb; kb += step) {
    const uint4 v = q[(int64_t)kb * 32];
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = kb * 64 + h * 32 + t * 8;
      const int grp = (kb * 64 + h * 32) / w.group;
      const float2 sc = scale2(s[grp * 8], w.fp16);
      const uint32_t zz = z == nullptr ? 0x0808u : z[grp * 8];
      const float z0 = (float)(zz & 255), z1 = (float)(zz >> 8);
      if (k >= w.k) continue;
      float a[8], b[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t u = words[2 * h + j];
        constexpr int pos[4] = {0, 4, 2, 6};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[4 * j + i] = (float)((u >> (4 * pos[i])) & 15) - z0;
          b[4 * j + i] = (float)((u >> (4 * pos[i] + 4)) & 15) - z1;
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4 xv = *reinterpret_cast<const uint4*>(x[m] + k);
        const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
        float da = 0.f, db = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x0 = bf16_lo(xw[i]), x1 = bf16_hi(xw[i]);
          da += a[2 * i] * x0 + a[2 * i + 1] * x1;
          db += b[2 * i] * x0 + b[2 * i + 1] * x1;
        }
        acc[m][0] += da * sc.x;
        acc[m][1] += db * sc.y;
      }
    }
  }
}

// number of an expert among those from e0 on; wraps to a large number for one that is not here
__device__ __forceinline__ unsigned local_expert(int32_t id, int e0) { return (unsigned)id - (unsigned)e0; }

constexpr int kDotWarps = 4;

// sums a tile's 16 rows over the lanes and warps of the CTA into red[row][m]
template <int MT>
__device__ __forceinline__ void tile_reduce(float (&acc)[MT][2], float (*red)[16][MT]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float v = acc[m][r];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if ((lane & 3) == 0) red[warp][(lane >> 2) + 8 * r][m] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * MT; i += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < kDotWarps; ++w) v += red[w][i / MT][i % MT];
    red[0][i / MT][i % MT] = v;
  }
  __syncthreads();
}

constexpr int kLinM = 4;

__global__ void __launch_bounds__(kDotWarps * 32)
w4_linear_kernel(W4Tensor w, const __nv_bfloat16* __restrict__ x, int64_t x_stride, int M,
                 const __nv_bfloat16* __restrict__ bias, __nv_bfloat16* __restrict__ out) {
  pdl_wait();
  pdl_launch();
  __shared__ float red[kDotWarps][16][kLinM];
  const int tile = blockIdx.x, m0 = blockIdx.y * kLinM;
  const __nv_bfloat16* rows[kLinM];
#pragma unroll
  for (int m = 0; m < kLinM; ++m) rows[m] = x + (int64_t)min(m0 + m, M - 1) * x_stride;
  float acc[kLinM][2] = {};
  tile_dot<kLinM>(w, tile, rows, threadIdx.x >> 5, kDotWarps, acc);
  tile_reduce<kLinM>(acc, red);
  for (int i = threadIdx.x; i < 16 * kLinM; i += blockDim.x) {
    const int m = i >> 4, n = tile * 16 + (i & 15);
    if (m0 + m < M && n < w.n) {
      const float b = bias == nullptr ? 0.f : __bfloat162float(bias[n]);
      out[(int64_t)(m0 + m) * w.n + n] = __float2bfloat16(red[0][i & 15][m] + b);
    }
  }
}

__device__ __forceinline__ float gated_act(float g, float u, int act) {
  if (act == 0) return g / (1.f + __expf(-g)) * u;
  if (act == 1) return 0.5f * g * (1.f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g))) * u;
  g = fminf(g, 7.f);
  u = fminf(fmaxf(u, -7.f), 7.f);
  return g / (1.f + __expf(-1.702f * g)) * (u + 1.f);
}

// a[pair] = act(gate) * up of the pair's expert; zeros for an expert that is not here
__global__ void __launch_bounds__(kDotWarps * 32)
w4_gate_up_kernel(W4Tensor w, int E, int e0, const __nv_bfloat16* __restrict__ x, int64_t x_stride, int topk,
                  const int32_t* __restrict__ ids, const __nv_bfloat16* __restrict__ bias, int act,
                  __nv_bfloat16* __restrict__ a, int a_stride) {
  pdl_wait();
  pdl_launch();
  __shared__ float red[kDotWarps][16][1];
  const int tile = blockIdx.x, pair = blockIdx.y, inter = w.n / 2;
  const unsigned e = local_expert(ids[pair], e0);
  if (e >= (unsigned)E) return;
  const __nv_bfloat16* rows[1] = {x + (int64_t)(pair / topk) * x_stride};
  float acc[1][2] = {};
  tile_dot<1>(w, (int64_t)e * w.tiles + tile, rows, threadIdx.x >> 5, kDotWarps, acc);
  tile_reduce<1>(acc, red);
  const int i = threadIdx.x, n = tile * 8 + i;
  if (i < 8 && n < inter) {
    float g = red[0][i][0], u = red[0][i + 8][0];
    if (bias != nullptr) {
      g += __bfloat162float(bias[(int64_t)e * w.n + n]);
      u += __bfloat162float(bias[(int64_t)e * w.n + inter + n]);
    }
    a[(int64_t)pair * a_stride + n] = __float2bfloat16(gated_act(g, u, act));
  }
}

__global__ void __launch_bounds__(kDotWarps * 32)
w4_down_kernel(W4Tensor w, int E, int e0, const __nv_bfloat16* __restrict__ a, int a_stride,
               const int32_t* __restrict__ ids, const __nv_bfloat16* __restrict__ bias, float* __restrict__ y) {
  pdl_wait();
  pdl_launch();
  __shared__ float red[kDotWarps][16][1];
  const int tile = blockIdx.x, pair = blockIdx.y;
  const unsigned e = local_expert(ids[pair], e0);
  if (e >= (unsigned)E) return;
  const __nv_bfloat16* rows[1] = {a + (int64_t)pair * a_stride};
  float acc[1][2] = {};
  tile_dot<1>(w, (int64_t)e * w.tiles + tile, rows, threadIdx.x >> 5, kDotWarps, acc);
  tile_reduce<1>(acc, red);
  const int n = tile * 16 + threadIdx.x;
  if (threadIdx.x < 16 && n < w.n)
    y[(int64_t)pair * w.n + n] =
        red[0][threadIdx.x][0] + (bias == nullptr ? 0.f : __bfloat162float(bias[(int64_t)e * w.n + n]));
}

__global__ void w4_combine_kernel(const float* __restrict__ y, const float* __restrict__ weights,
                                  const int32_t* __restrict__ ids, int E, int e0, int topk, int H,
                                  __nv_bfloat16* __restrict__ out) {
  pdl_wait();
  pdl_launch();
  const int t = blockIdx.x;
  for (int c = threadIdx.x; c < H; c += blockDim.x) {
    float v = 0.f;
    for (int j = 0; j < topk; ++j) {
      if (local_expert(ids[(int64_t)t * topk + j], e0) < (unsigned)E) v += weights[(int64_t)t * topk + j] * y[((int64_t)t * topk + j) * H + c];
    }
    out[(int64_t)t * H + c] = __float2bfloat16(v);
  }
}

W4Tensor tensor_of(const MsglW4* w) {
  return {(const uint4*)w->q, (const uint32_t*)w->s, (const uint16_t*)w->z, w->tiles, w->kb, w->kg, w->group,
          w->n, w->k, w->fp16};
}

}  // namespace

extern "C" int msgl_w4_linear(void* out, const void* x, int64_t x_stride, int M, const MsglW4* w, const void* bias,
                              cudaStream_t s) {
  if (M == 0 || w->n == 0) return 0;
  const cudaError_t e =
      msgl_launch(w4_linear_kernel, dim3(w->tiles, (M + kLinM - 1) / kLinM), dim3(kDotWarps * 32), 0, s, 1,
                  tensor_of(w), (const __nv_bfloat16*)x, x_stride, M, (const __nv_bfloat16*)bias, (__nv_bfloat16*)out);
  return e == cudaSuccess ? 0 : 4;
}

extern "C" int64_t msgl_w4_experts_workspace(int T, int topk, const MsglW4* w1, const MsglW4* w2) {
  const int64_t pairs = (int64_t)T * topk;
  return pairs * w2->kb * 64 * 2 + pairs * w2->n * 4;
}

extern "C" int msgl_w4_experts(void* out, const void* x, int64_t x_stride, int T, int topk, const MsglW4* w1,
                               const MsglW4* w2, int E, int e0, const float* weights, const int32_t* ids,
                               const void* b1, const void* b2, int act, void* workspace, cudaStream_t s) {
  if (T == 0) return 0;
  const int pairs = T * topk, a_stride = w2->kb * 64;
  __nv_bfloat16* a = (__nv_bfloat16*)workspace;
  float* y = (float*)((uint8_t*)workspace + (int64_t)pairs * a_stride * 2);
  cudaError_t e = msgl_launch(w4_gate_up_kernel, dim3(w1->tiles, pairs), dim3(kDotWarps * 32), 0, s, 1, tensor_of(w1),
                              E, e0, (const __nv_bfloat16*)x, x_stride, topk, ids, (const __nv_bfloat16*)b1, act, a,
                              a_stride);
  if (e == cudaSuccess)
    e = msgl_launch(w4_down_kernel, dim3(w2->tiles, pairs), dim3(kDotWarps * 32), 0, s, 1, tensor_of(w2), E, e0,
                    (const __nv_bfloat16*)a, a_stride, ids, (const __nv_bfloat16*)b2, y);
  if (e == cudaSuccess)
    e = msgl_launch(w4_combine_kernel, dim3(T), dim3(256), 0, s, 1, (const float*)y, weights, ids, E, e0, topk, w2->n,
                    (__nv_bfloat16*)out);
  return e == cudaSuccess ? 0 : 4;
}
