// The 4-bit linear product out [M, N] = x [M, K] w^T (+ bias); see w4.cuh for the weights' layout and
// the streaming product.
//
// Few tokens: persistent CTAs of 16 warps, one per SM. With `splits` > 1 a cluster of that many CTAs
// shares its tiles and cuts the inputs: each CTA reads its share of the activations only, and the sums
// meet through distributed shared memory. The split is the one whose largest share of weights, plus the
// activations that every CTA reads, is smallest (plan()).
#include <algorithm>
#include <mutex>

#include "w4.cuh"

using namespace msgl;

namespace {

struct LinearArgs {
  W4Tensor w;
  const __nv_bfloat16* x;
  int64_t x_stride;
  int M;
  const __nv_bfloat16* bias;
  __nv_bfloat16* out;
  int splits, max_tiles;
};

template <int NT, int G, bool Z>
__global__ void __launch_bounds__(kW4Threads, 1) w4_linear_kernel(const __grid_constant__ LinearArgs p) {
  using C = W4Chunk<G>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int clusters = gridDim.x / p.splits, cl = blockIdx.x / p.splits, rank = blockIdx.x % p.splits;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int t0 = (int)((int64_t)p.w.tiles * cl / clusters), t1 = (int)((int64_t)p.w.tiles * (cl + 1) / clusters);
  const int chunks = p.w.kb / C::kUnits;
  const int c0 = chunks * rank / p.splits, nc = chunks * (rank + 1) / p.splits - c0;
  float4* part = reinterpret_cast<float4*>(smem);
  float4* sums = reinterpret_cast<float4*>(smem + w4_part_bytes<NT>());  // [max_tiles][NT][32] with splits
  const int sum_bytes = p.splits > 1 ? p.max_tiles * NT * 512 : 0;
  uint8_t* xs = smem + w4_part_bytes<NT>() + sum_bytes;
  const int kn = nc * C::kUnits * 64, pitch = w4_pitch(kn);

  pdl_launch();
  // the weights do not depend on earlier kernels' results, but may have been written by one: they may be
  // brought into L2 before the wait, not read
  if (lane == 0 && t1 > t0) {
    const int64_t total = (int64_t)(t1 - t0) * nc;
    const int a = (int)(total * warp / kW4Warps), b = (int)(total * (warp + 1) / kW4Warps);
    const int n = min(min(b - a, nc - a % nc), C::kDepth * 2);
    if (n > 0)
      prefetch_l2(p.w.q + ((int64_t)(t0 + a / nc) * p.w.kb + (c0 + a % nc) * C::kUnits) * 32, n * C::kUnits * 512);
  }
  pdl_wait();
  if (t1 == t0) return;  // the same for every CTA of a cluster

  const auto store = [&](int tile, const float (&acc)[NT][4]) {
    const int n = (t0 + tile) * 16 + g;
    const float b0 = p.bias != nullptr && n < p.w.n ? __bfloat162float(p.bias[n]) : 0.f;
    const float b1 = p.bias != nullptr && n + 8 < p.w.n ? __bfloat162float(p.bias[n + 8]) : 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int m = nt * 8 + 2 * t + c;
        if (m >= p.M) continue;
        __nv_bfloat16* o = p.out + (int64_t)m * p.w.n + n;
        if (n < p.w.n) o[0] = __float2bfloat16(acc[nt][c] + b0);
        if (n + 8 < p.w.n) o[8] = __float2bfloat16(acc[nt][2 + c] + b1);
      }
  };
  const auto load = [&] {
    load_rows(xs, pitch, p.M, c0 * C::kUnits * 64, kn, p.w.k, [&](int r) { return p.x + (int64_t)r * p.x_stride; });
  };
  if (p.splits == 1) {
    run_tiles<NT, G, Z>(p.w, t0, t1 - t0, c0, nc, xs, pitch, p.M, part, load, store);
    return;
  }
  run_tiles<NT, G, Z>(p.w, t0, t1 - t0, c0, nc, xs, pitch, p.M, part, load, [&](int tile, const float (&acc)[NT][4]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      sums[(tile * NT + nt) * 32 + lane] = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
  });
  cluster_sync();
  for (int tile = rank * kW4Warps + warp; tile < t1 - t0; tile += p.splits * kW4Warps) {
    float acc[NT][4] = {};
    for (int r = 0; r < p.splits; ++r) {
      const uint32_t from = dsmem_addr(smem_u32(sums + (tile * NT) * 32 + lane), r);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float4 v = ld_dsmem_v4(from + nt * 512);
        acc[nt][0] += v.x, acc[nt][1] += v.y, acc[nt][2] += v.z, acc[nt][3] += v.w;
      }
    }
    store(tile, acc);
  }
  cluster_sync();  // the other CTAs of the cluster read this one's shared memory
}

constexpr int kSmemMax = 227 * 1024;

struct Plan {
  int splits, grid, max_tiles, smem;
};

// CTAs of a cluster of `splits` that run at once, in whole clusters (148 SMs, not all in groups of 8)
template <auto Kernel>
int resident_ctas(int splits) {
  static std::mutex mu;
  static int known[64][9] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> guard(mu);
  int& k = known[dev][splits];
  if (k != 0) return k;
  if (splits == 1) return k = msgl_num_sms();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits);
  cfg.blockDim = dim3(kW4Threads);
  cfg.dynamicSmemBytes = kSmemMax;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, Kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = 1;
  }
  return k = n * splits;
}

// The split of the inputs with the least estimated time: the largest CTA's weight bytes at an SM's
// share of the memory rate (43 B/ns), its activations at the L2's (four times that), and 1.5 us for the
// exchange. Returns splits = 0 if the rows do not fit.
template <auto Kernel, int NT, int G>
Plan plan(const W4Tensor& w, int M) {
  const int chunks = w.kb / W4Chunk<G>::kUnits;
  Plan best = {0, 0, 0, 0};
  double best_ns = 1e30;
  for (int s = 1; s <= 8; s *= 2) {
    if (s > chunks) break;
    const int clusters = std::min(resident_ctas<Kernel>(s) / s, w.tiles);
    if (clusters < 1) continue;
    const int tiles = (w.tiles + clusters - 1) / clusters;
    const int kn = (chunks + s - 1) / s * W4Chunk<G>::kUnits * 64;
    const int64_t smem = w4_part_bytes<NT>() + (s > 1 ? (int64_t)tiles * NT * 512 : 0) + (int64_t)M * w4_pitch(kn);
    if (smem > kSmemMax) continue;
    const double ns = tiles * (kn / 64) * 512.0 / 43 + M * kn * 2.0 / 172 + (s > 1 ? 1500 : 0);
    if (ns < best_ns) {
      best_ns = ns;
      best = {s, clusters * s, tiles, (int)smem};
    }
  }
  return best;
}

template <int NT, int G, bool Z>
int launch_linear(LinearArgs p, cudaStream_t s) {
  constexpr auto kernel = w4_linear_kernel<NT, G, Z>;
  if (msgl_set_smem<kernel>(kSmemMax) != cudaSuccess) return 4;
  const Plan pl = plan<kernel, NT, G>(p.w, p.M);
  if (pl.splits == 0) return 3;
  p.splits = pl.splits;
  p.max_tiles = pl.max_tiles;
  return msgl_launch(kernel, dim3(pl.grid), dim3(kW4Threads), pl.smem, s, pl.splits, p) == cudaSuccess ? 0 : 4;
}

template <int NT>
int launch_linear_nt(const LinearArgs& p, cudaStream_t s) {
  const bool z = p.w.z != nullptr;
  switch (p.w.group) {
    case 32: return z ? launch_linear<NT, 32, true>(p, s) : launch_linear<NT, 32, false>(p, s);
    case 64: return z ? launch_linear<NT, 64, true>(p, s) : launch_linear<NT, 64, false>(p, s);
    default: return z ? launch_linear<NT, 128, true>(p, s) : launch_linear<NT, 128, false>(p, s);
  }
}

// rows in one launch if their activations fit into shared memory, else in halves
int linear_rows(const LinearArgs& p, cudaStream_t s) {
  const int rc = p.M <= 8 ? launch_linear_nt<1>(p, s) : p.M <= 16 ? launch_linear_nt<2>(p, s) : launch_linear_nt<4>(p, s);
  if (rc != 3 || p.M == 1) return rc;
  LinearArgs a = p, b = p;
  a.M = p.M > 16 ? 16 : p.M > 8 ? 8 : p.M / 2;
  b.M = p.M - a.M;
  b.x += a.M * p.x_stride;
  b.out += (int64_t)a.M * p.w.n;
  const int ra = linear_rows(a, s);
  return ra != 0 ? ra : linear_rows(b, s);
}

}  // namespace

extern "C" int msgl_w4_linear(void* out, const void* x, int64_t x_stride, int M, const MsglW4* w, const void* bias,
                              cudaStream_t s) {
  if (M == 0) return 0;
  LinearArgs p = {w4_tensor(w), (const __nv_bfloat16*)x, x_stride, M, (const __nv_bfloat16*)bias, (__nv_bfloat16*)out,
                  1, 0};
  for (int m = 0; m < M; m += 32) {
    LinearArgs a = p;
    a.M = std::min(32, M - m);
    a.x += m * x_stride;
    a.out += (int64_t)m * w->n;
    const int rc = linear_rows(a, s);
    if (rc != 0) return rc;
  }
  return 0;
}
