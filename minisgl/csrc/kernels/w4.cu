// The 4-bit linear product out [M, N] = x [M, K] w^T (+ bias); see w4.cuh for the weights' layout and
// the streaming product.
//
// Few tokens: persistent CTAs, one per SM. With `splits` > 1 a cluster of that many CTAs
// shares its tiles and cuts the inputs: each CTA reads its share of the activations only, and the sums
// meet through distributed shared memory. The split is the one whose largest share of weights, plus the
// activations that every CTA reads, is smallest (plan()).
#include <algorithm>
#include <atomic>

#include "w4_gemm.cuh"

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

template <int NT, int G, bool Z, bool F>
__global__ void __launch_bounds__(w4_threads<NT>(), 1) w4_linear_kernel(const __grid_constant__ LinearArgs p) {
  using R = W4Record<G, Z>;
  constexpr int kWarps = w4_warps<NT>(), kRun = w4_run_bytes<NT, G, Z>();
  extern __shared__ __align__(16) uint8_t smem[];
  const int clusters = gridDim.x / p.splits, cl = blockIdx.x / p.splits, rank = blockIdx.x % p.splits;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int t0 = p.w.tiles / clusters * cl + min(cl, p.w.tiles % clusters);
  const int t1 = t0 + p.w.tiles / clusters + (cl < p.w.tiles % clusters ? 1 : 0);
  const int c0 = p.w.kc * rank / p.splits, nc = p.w.kc * (rank + 1) / p.splits - c0;
  float4* sums = reinterpret_cast<float4*>(smem + kRun);  // [max_tiles][2 NT][32] with splits
  uint8_t* xs = smem + kRun + (p.splits > 1 ? p.max_tiles * NT * 1024 : 0);
  const int pitch = w4_pitch(nc * 128);
  W4Runs<NT, G, Z, F> runs{smem};

  pdl_launch();
  // the weights do not depend on earlier kernels' results, but may have been written by one: they may be
  // brought into L2 before the wait, not read
  if (lane == 0) {
    const int total = (t1 - t0) * nc, a = runs.bound(total, warp), n = min(runs.bound(total, warp + 1) - a, kW4Slots);
    if (n > 0 && a % nc + n <= nc)
      prefetch_l2(p.w.data + ((int64_t)(t0 + a / nc) * p.w.kc + c0 + a % nc) * R::kBytes, n * R::kBytes);
  }
  runs.init();
  __syncthreads();
  pdl_wait();

  const auto store = [&](int tile, const float (&acc)[2][NT][4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // rows g, g + 8, g + 16, g + 24 of the tile
      const int n = (t0 + tile) * 32 + r * 8 + g;
      if (n >= p.w.n) continue;
      const float b = p.bias != nullptr ? __bfloat162float(p.bias[n]) : 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int m = nt * 8 + 2 * t + c;
          if (m < p.M) p.out[(int64_t)m * p.w.n + n] = __float2bfloat16(acc[r >> 1][nt][2 * (r & 1) + c] * kW4Unit + b);
        }
    }
  };
  const auto row = [&](int r) { return p.x + (int64_t)r * p.x_stride; };
  if (p.splits == 1) {
    runs.template run<false>(p.w, t0, t1 - t0, c0, nc, xs, pitch, p.M, row, store);
    return;
  }
  runs.template run<true>(p.w, t0, t1 - t0, c0, nc, xs, pitch, p.M, row, [&](int tile, const float (&acc)[2][NT][4]) {
    W4Runs<NT, G, Z, F>::put(sums + tile * NT * 64 + lane, acc);
  });
  cluster_sync();
  for (int tile = rank * kWarps + warp; tile < t1 - t0; tile += p.splits * kWarps) {
    float acc[2][NT][4] = {};
    for (int r = 0; r < p.splits; ++r) {
      const uint32_t from = dsmem_addr(smem_u32(sums + tile * NT * 64 + lane), r);
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) {
        const float4 v = ld_dsmem_v4(from + i * 512);
        float(&o)[4] = acc[i / NT][i % NT];
        o[0] += v.x, o[1] += v.y, o[2] += v.z, o[3] += v.w;
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

// The split of the inputs with the least estimated time: the largest CTA's weight bytes at an SM's
// share of the memory rate (43 B/ns), its activations at the L2's (four times that), and 1.5 us for the
// exchange. It ranks splits and is no forecast: the products' issue slots are not in it (16 x 5120 x 17408, groups of
// 64 with zero points: 9.9 us estimated, 23 measured; there only a split in 8 has room for the rows). Returns splits = 0
// if the rows do not fit.
template <auto Kernel, int NT, int G, bool Z>
Plan plan(const W4Tensor& w, int M) {
  Plan best = {0, 0, 0, 0};
  double best_ns = 1e30;
  for (int s = 1; s <= 8 && s <= w.kc; s *= 2) {
    const int clusters = std::min(w4_resident_clusters<Kernel>(s, w4_threads<NT>()), w.tiles);
    if (clusters < 1) continue;
    const int tiles = (w.tiles + clusters - 1) / clusters;
    const int records = (w.kc + s - 1) / s, kn = records * 128;
    const int64_t smem = w4_run_bytes<NT, G, Z>() + (s > 1 ? (int64_t)tiles * NT * 1024 : 0) + (int64_t)M * w4_pitch(kn);
    if (smem > kSmemMax) continue;
    const double ns = (double)tiles * records * W4Record<G, Z>::kBytes / 43 + M * kn * 2.0 / 172 + (s > 1 ? 1500 : 0);
    if (ns < best_ns) {
      best_ns = ns;
      best = {s, clusters * s, tiles, (int)smem};
    }
  }
  return best;
}

template <int NT, int G, bool Z, bool F>
int launch_linear(LinearArgs p, cudaStream_t s) {
  constexpr auto kernel = w4_linear_kernel<NT, G, Z, F>;
  if (msgl_set_smem<kernel>(kSmemMax) != cudaSuccess) return 4;
  const Plan pl = plan<kernel, NT, G, Z>(p.w, p.M);
  if (pl.splits == 0) return 3;
  p.splits = pl.splits;
  p.max_tiles = pl.max_tiles;
  return w4_launch(kernel, dim3(pl.grid), dim3(w4_threads<NT>()), pl.smem, s, pl.splits, p) == cudaSuccess ? 0 : 4;
}

template <int NT>
int launch_linear_nt(const LinearArgs& p, const MsglW4* w, cudaStream_t s) {
  return w4_dispatch(w, [&](auto g, auto z, auto f) { return launch_linear<NT, g(), z(), f()>(p, s); });
}

// Tokens up to which the streaming product is taken (one or two columns of 8).
constexpr int kStreamTokens = 16;

// rows in one launch if their activations fit into shared memory, else in parts; 3 if not one row does
int linear_rows(const LinearArgs& p, const MsglW4* w, cudaStream_t s) {
  const int rc = p.M <= 8 ? launch_linear_nt<1>(p, w, s) : launch_linear_nt<2>(p, w, s);
  if (rc != 3 || p.M == 1) return rc;
  LinearArgs a = p, b = p;
  a.M = p.M > 8 ? 8 : p.M / 2;
  b.M = p.M - a.M;
  b.x += a.M * p.x_stride;
  b.out += (int64_t)a.M * p.w.n;
  const int ra = linear_rows(a, w, s);
  return ra != 0 ? ra : linear_rows(b, w, s);
}

// Form override for tests (0, 0: by the estimate): halves of a tile and cuts of the inputs. Not for concurrent use.
std::atomic<int> g_halves{0}, g_splits{0};

// many tokens: tiles of 128 or 256 rows by up to 208 tokens; where these leave SMs idle a cluster cuts the inputs
int linear_tiles(const LinearArgs& a, const MsglW4* w, cudaStream_t s) {
  W4GemmArgs p = {};
  p.w = a.w;
  p.group = w->group, p.zeros = w->zeros, p.fp16 = w->fp16;
  p.in = a.x, p.in_stride = a.x_stride;
  p.bias = a.bias;
  p.out = a.out, p.out_stride = w->n;
  p.M = a.M;
  p.m_tiles = (a.M + kGwMaxTokens - 1) / kGwMaxTokens;
  p.bn = ((a.M + p.m_tiles - 1) / p.m_tiles + 15) / 16 * 16;
  p.m_tiles = (a.M + p.bn - 1) / p.bn;
  // Halves of a tile and cuts of the inputs with the least estimated time, in clocks per 128 inputs of a tile:
  // conversion 450 a half (measured with bf16 scales; fp16 ones take about a quarter longer), the tensor core 4 a token and
  // half, the tokens' rows from L2 5 a token; the exchange 2000 and 20 a token and half.
  double best = 1e30;
  int halves = 1;
  const int only_h = g_halves.load(), only_s = g_splits.load();
  for (int h = 1; h <= 2; ++h) {
    if (only_h != 0 && h != only_h) continue;
    const int64_t units = (int64_t)((a.w.tiles + 4 * h - 1) / (4 * h)) * p.m_tiles;
    if (units >= (1ll << 31)) return 3;
    for (int s = 1; s <= std::min(8, a.w.kc); ++s) {
      if (only_s != 0 && s != only_s) continue;
      if (s > 1 && p.bn * h * 512 > kGwRoom) continue;  // the fp32 tile does not fit
      const int at_once = h == 2 ? w4_gemm_clusters<2>(s) : w4_gemm_clusters<1>(s);
      if (at_once < 1) continue;
      const double waves = (double)((units + at_once - 1) / at_once), records = (a.w.kc + s - 1) / s;
      const double per = std::max({450.0 * h, 4.0 * p.bn * h, 5.0 * p.bn});
      const double t = waves * (records * per + 1500) + (s > 1 ? 2000 + 20.0 * p.bn * h : 0);
      if (t < best) best = t, halves = h, p.splits = s;
    }
  }
  if (p.splits == 0) return 3;
  p.n_tiles = (a.w.tiles + 4 * halves - 1) / (4 * halves);
  const int64_t units = (int64_t)p.n_tiles * p.m_tiles;
  if (p.splits > 1) {
    const int grid = (int)(units * p.splits);
    return halves == 2 ? w4_gemm_launch<kW4Dense, 2, true>(p, grid, s) : w4_gemm_launch<kW4Dense, 1, true>(p, grid, s);
  }
  const int grid = (int)std::min<int64_t>(units, msgl_num_sms());
  return halves == 2 ? w4_gemm_launch<kW4Dense, 2, false>(p, grid, s) : w4_gemm_launch<kW4Dense, 1, false>(p, grid, s);
}

}  // namespace

extern "C" int msgl_w4_linear(void* out, const void* x, int64_t x_stride, int M, const MsglW4* w, const void* bias,
                              int* launches, cudaStream_t s) {
  *launches = w4_launched = 0;
  if (M == 0) return 0;
  const LinearArgs p = {w4_tensor(w), (const __nv_bfloat16*)x, x_stride, M, (const __nv_bfloat16*)bias,
                        (__nv_bfloat16*)out, 1, 0};
  int rc = M <= kStreamTokens ? linear_rows(p, w, s) : 3;
  if (rc == 3) rc = linear_tiles(p, w, s);
  *launches = w4_launched;
  return rc;
}

extern "C" void msgl_w4_force_form(int halves, int splits) { g_halves.store(halves), g_splits.store(splits); }

MSGL_ERROR_ACCESSOR(msgl_err_w4)
