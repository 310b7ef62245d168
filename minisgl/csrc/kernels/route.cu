// Expert routing with softmax or sigmoid scores, a balancing bias, expert groups, top-k and
// renormalised weights.
//
//   p = softmax(l) or sigmoid(l)            the score of every expert
//   v = p + bias (without a bias: l)        what the choice goes by
//   rank(group) = max v, or the sum of its two best p + bias; the best `kept` groups stay
//   ids = the k largest v of the experts that stay, largest first, equal ones by their number
//   w = p[ids] (/ sum of p[ids]) * scale
//
// A NaN logit counts as -inf and +inf as the largest float; a row without a finite logit has scores of
// zero, and weights whose sum is zero stay zero. Biases are held to the floats' finite range (NaN: the
// lowest), so every v is finite and the order is total.
#include <cfloat>

#include "api.h"
#include "common.cuh"

using namespace msgl;

namespace {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxE = 512;

template <typename T>
__device__ __forceinline__ float logit_of(const T* p);
template <>
__device__ __forceinline__ float logit_of<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float logit_of<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }

__device__ __forceinline__ float clean_logit(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }
__device__ __forceinline__ float clean_bias(float b) { return b != b ? -FLT_MAX : fmaxf(fminf(b, FLT_MAX), -FLT_MAX); }

// largest value of the warp's lanes, then the lowest index that has it
__device__ __forceinline__ void warp_best(double& v, int& i) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, i, o);
    if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
  }
}

// One warp per token, everything in 64 bits.
template <typename T>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_experts_kernel(const T* __restrict__ logits, int64_t stride, const float* __restrict__ bias, int n_tok, int E,
                     int topk, int sigmoid, int groups, int kept, int top2, int renorm, float scale,
                     float* __restrict__ weights, int32_t* __restrict__ ids) {
  pdl_wait();
  pdl_launch();
  extern __shared__ double route_sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * kRouteWarps + warp;
  if (t >= n_tok) return;
  double* p = route_sm + (size_t)warp * 2 * E;  // scores
  double* v = p + E;                            // what the choice goes by
  const T* row = logits + (int64_t)t * stride;
  const bool by_logit = bias == nullptr;

  double mx = -INFINITY;
  for (int e = lane; e < E; e += 32) {
    const double x = clean_logit(logit_of(row + e));
    p[e] = x;
    mx = fmax(mx, x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  double sum = 0.0;
  for (int e = lane; e < E; e += 32) {
    const double x = p[e];
    double s;
    if (sigmoid) s = 1.0 / (1.0 + exp(-x));
    else s = mx == -INFINITY ? 0.0 : exp(x - mx);
    v[e] = by_logit ? fmax(x, -(double)FLT_MAX * 2) : (double)clean_bias(bias[e]);
    p[e] = s;
    sum += s;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  for (int e = lane; e < E; e += 32) {
    if (!sigmoid) p[e] = sum > 0.0 ? p[e] / sum : 0.0;
    if (!by_logit) v[e] += p[e];
  }
  __syncwarp();

  if (groups > 1) {
    const int per = E / groups;
    // ranks of up to 256 groups: lane g, g + 32, ...
    double rank[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int g = lane + 32 * i;
      if (g >= groups) { rank[i] = -INFINITY; continue; }
      double a = -INFINITY, b = -INFINITY;
      for (int j = 0; j < per; ++j) {
        const double x = (by_logit && top2) ? p[g * per + j] : v[g * per + j];
        if (x > a) { b = a; a = x; } else if (x > b) b = x;
      }
      rank[i] = top2 ? a + b : a;
    }
    unsigned keep = 0;  // bit i: this lane's group lane + 32 i stays
    for (int n = 0; n < kept; ++n) {
      double bv = -INFINITY;
      int bi = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (rank[i] > bv) { bv = rank[i]; bi = lane + 32 * i; }
      warp_best(bv, bi);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane + 32 * i == bi) { rank[i] = -INFINITY; keep |= 1u << i; }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int g = lane + 32 * i;
      if (g < groups && !((keep >> i) & 1))
        for (int j = 0; j < per; ++j) v[g * per + j] = -INFINITY;
    }
    __syncwarp();
  }

  double total = 0.0;
  for (int n = 0; n < topk; ++n) {
    double bv = -INFINITY;
    int bi = 0x7fffffff;
    for (int e = lane; e < E; e += 32)
      if (v[e] > bv) { bv = v[e]; bi = e; }
    warp_best(bv, bi);
    total += p[bi];
    if (lane == 0) {
      ids[(int64_t)t * topk + n] = bi;
      v[bi] = -INFINITY;
    }
    __syncwarp();
  }
  if (lane < topk) {
    const double w = p[ids[(int64_t)t * topk + lane]];
    weights[(int64_t)t * topk + lane] = (float)((renorm ? (total > 0.0 ? w / total : 0.0) : w) * (double)scale);
  }
}

}  // namespace

extern "C" int msgl_route_experts(const void* logits, int is_fp32, int64_t stride, const float* bias, int n_tok, int E,
                                  int topk, int sigmoid, int groups, int kept, int top2, int renorm, float scale,
                                  float* weights, int32_t* ids, cudaStream_t s) {
  if (n_tok == 0) return 0;
  if (E < 1 || E > kRouteMaxE || topk < 1 || topk > 32 || groups < 1 || groups > 256 || E % groups != 0) return 3;
  const dim3 grid((n_tok + kRouteWarps - 1) / kRouteWarps), block(kRouteWarps * 32);
  const size_t smem = (size_t)kRouteWarps * 2 * E * sizeof(double);
  const cudaError_t e =
      is_fp32 ? msgl_launch(route_experts_kernel<float>, grid, block, smem, s, 1, (const float*)logits, stride, bias,
                            n_tok, E, topk, sigmoid, groups, kept, top2, renorm, scale, weights, ids)
              : msgl_launch(route_experts_kernel<__nv_bfloat16>, grid, block, smem, s, 1,
                            (const __nv_bfloat16*)logits, stride, bias, n_tok, E, topk, sigmoid, groups, kept, top2,
                            renorm, scale, weights, ids);
  return e == cudaSuccess ? 0 : 4;
}
