// The experts' products of an MoE layer with 4-bit weights (layout and streaming product in w4.cuh):
//   a[p] = act(w1[e] x[token]) for every (token, choice) pair p, y[p] = w2[e] a[p], out = sum of weight * y.
//
// Few tokens: the chosen experts' tiles, one after another, are cut into equal runs, one per SM. Every CTA
// counts the pairs per expert itself (they are few) instead of waiting for a kernel that would, so a
// layer is three launches; the counting of the second product overlaps the end of the first. The
// activated values between the products are two bf16 each, 16 bits, whose columns are mostly there anyway (in one, their
// rounding put the result 0.0024 off in the 2-norm, where its own rounding is 0.0017); y is fp32 and the sum over a
// token's experts runs in the order of its choices, so results do not vary.
//
// Many tokens: a kernel sorts the pairs by expert and lists tiles of up to 64 or 128 of an expert's pairs; the products
// run on the tensor core (w4_gemm.cuh), the first one gathering the tokens' rows, and the sum is the same.
//
// 128 experts of 2048 x 768, 8 a token, groups of 128, whole layer: 1 token 17.9 us (3.0 for the bytes; three launches
// of 5 to 7 us), 16 tokens 51 (25), 128 tokens 113 (45); on the tensor core 256 tokens 156 (47), 512 tokens 181 (48),
// 2048 tokens 400 (92), 16384 tokens 2640 (737), of which the one block that sorts the 131072 pairs takes 96 (15 at 2048
// tokens, 7 at 512).
#include <algorithm>

#include "w4_gemm.cuh"

using namespace msgl;

namespace {

constexpr int kMoeMaxPairs = 4096;  // of the streaming product: their experts are kept in shared memory
constexpr int kMoeMaxExperts = 1024;
constexpr int kSmemMax = 227 * 1024;

// number of an expert among those from e0 on; wraps to a large number for one that is not here
MSGL_DEVICE unsigned local_expert(int32_t id, int e0) { return (unsigned)id - (unsigned)e0; }

// shared memory of the lists behind the runs', a multiple of 16
__host__ __device__ inline int prelude_bytes(int E, int pairs, int rows) {
  return (16 + 32 + 2 * E + pairs / rows + pairs + 3) / 4 * 16;
}

struct ExpertArgs {
  W4Tensor w;
  int E, e0, pairs, topk;
  const int32_t* ids;
  const __nv_bfloat16* in;  // rows of x (gated: token pair / topk) or of the activated values (pair; two planes, w4_act_parts)
  int64_t in_stride;
  const __nv_bfloat16* bias;  // [E, n]
  __nv_bfloat16* a;           // gated: [2, pairs, a_stride]
  float* y;                   // else: [pairs, n]
  int a_stride, act, rows;    // rows: pairs of one pass
};

// columns that a pair takes of the streaming product: the second product has its activated values in two parts, side by
// side, and adds their sums
constexpr int columns_of(bool gated) { return gated ? 1 : 2; }

template <int NT, int G, bool Z, bool F, bool GATED>
__global__ void __launch_bounds__(w4_threads<NT>(), 1) w4_experts_kernel(const __grid_constant__ ExpertArgs p) {
  using R = W4Record<G, Z>;
  constexpr int kWarps = w4_warps<NT>(), kThreads = w4_threads<NT>();
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // units: up to p.rows of an expert's pairs
  int* const list = reinterpret_cast<int*>(smem + w4_run_bytes<NT, G, Z>());  // [16] pairs of the unit at hand
  int* const seen = list + 16;                            // [32] warps' counts
  int* const count = seen + 32;                           // [E] pairs of every expert
  int* const units = count + p.E;                         // [E + pairs / rows] expert, number of the unit in it
  uint32_t* const lid = reinterpret_cast<uint32_t*>(units + p.E + p.pairs / p.rows);  // [pairs] experts here
  uint8_t* xs = smem + (w4_run_bytes<NT, G, Z>() + prelude_bytes(p.E, p.pairs, p.rows));
  W4Runs<NT, G, Z, F> runs{smem};
  runs.init();

  // The second product's ids were complete before the first product's kernel began its work, which is
  // before this kernel could start (it triggers its dependents after its own wait).
  if constexpr (GATED) pdl_wait();
  pdl_launch();
  // Up to 32 pairs are a lane each: the lanes that hold an expert first stand for its unit, if none has more pairs
  // than fit one (decoding a few tokens; the lists below cost 2 us there).
  unsigned my_e = 0xffffffffu, same = 0, leaders = 0;
  bool few = p.pairs <= 32;
  if (few) {
    if (lane < p.pairs) my_e = local_expert(p.ids[lane], p.e0);
    same = __match_any_sync(0xffffffffu, my_e);
    leaders = __ballot_sync(0xffffffffu, my_e < (unsigned)p.E && __ffs(same) == lane + 1);
    few = !__any_sync(0xffffffffu, my_e < (unsigned)p.E && __popc(same) > p.rows);
  }
  // the lane that stands for unit `un`
  const auto leader_of = [&](int un) {
    const bool is = ((leaders >> lane) & 1) && __popc(leaders & ((1u << lane) - 1)) == un;
    return __ffs(__ballot_sync(0xffffffffu, is)) - 1;
  };
  int n_units = __popc(leaders);
  if (!few) {
    n_units = 0;
    for (int e = threadIdx.x; e < p.E; e += kThreads) count[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.pairs; i += kThreads) {
      const unsigned e = local_expert(p.ids[i], p.e0);
      lid[i] = e;
      if (e < (unsigned)p.E) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    // the units, expert by expert: sums of 32 experts a warp, then of the warps
    for (int b = 0; b < p.E; b += kThreads) {
      const int e = b + (int)threadIdx.x, mine = e < p.E ? (count[e] + p.rows - 1) / p.rows : 0;
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      if (lane == 31) seen[warp] = sum;
      __syncthreads();
      int before = lane < kWarps ? seen[lane] : 0;
      const int all = __reduce_add_sync(0xffffffffu, before);
      before = __reduce_add_sync(0xffffffffu, lane < warp ? before : 0);
      for (int i = 0; i < mine; ++i) units[n_units + before + sum - mine + i] = e | i << 16;
      n_units += all;
      if (b + kThreads < p.E) __syncthreads();  // seen is used again
    }
  }
  __syncthreads();
  // this CTA's run of the units' tiles: an equal share, whichever experts it falls on
  const int all = n_units * p.w.tiles, share = all / (int)gridDim.x, rest = all % (int)gridDim.x;
  int pos = (int)blockIdx.x * share + min((int)blockIdx.x, rest);
  const int end = pos + share + ((int)blockIdx.x < rest ? 1 : 0);
  const int pitch = w4_pitch(p.w.kc * 128);
  if constexpr (!GATED) {
    // bring the run's first weights into L2 while the first product ends
    const int un = pos / p.w.tiles;
    const int e = pos >= end ? 0 : few ? (int)__shfl_sync(0xffffffffu, my_e, leader_of(un)) : units[un] & 0xffff;
    if (lane == 0 && pos < end) {
      const int ta = pos - un * p.w.tiles, nt = min(p.w.tiles - ta, end - pos);
      const int64_t tile = (int64_t)e * p.w.tiles + ta;
      const int a = runs.bound(nt * p.w.kc, warp), n = min(runs.bound(nt * p.w.kc, warp + 1) - a, kW4Slots);
      if (n > 0) prefetch_l2(p.w.data + (tile * p.w.kc + a) * R::kBytes, n * R::kBytes);
    }
    pdl_wait();
  }

  // the pairs are looked through by all warps, a run of whole 32s each
  const int per = ((p.pairs + 31) / 32 + kWarps - 1) / kWarps * 32;
  while (pos < end) {
    const int un = pos / p.w.tiles, ta = pos - un * p.w.tiles, nt = min(p.w.tiles - ta, end - pos);
    int e, nx;
    __syncthreads();  // the previous unit's list is done with
    if (few) {
      const int leader = leader_of(un);
      const unsigned m = __shfl_sync(0xffffffffu, same, leader);
      e = __shfl_sync(0xffffffffu, my_e, leader);
      nx = __popc(m);
      if (warp == 0 && ((m >> lane) & 1)) list[__popc(m & ((1u << lane) - 1))] = lane;
    } else {
      const int unit = units[un], i0 = unit >> 16;
      e = unit & 0xffff;
      // the expert's pairs are cut into equal units; every CTA finds the same ones in the same order
      const int c = count[e], cuts = c <= p.rows ? 1 : (c + p.rows - 1) / p.rows;
      const int m0 = cuts == 1 ? 0 : c * i0 / cuts;
      nx = (cuts == 1 ? c : c * (i0 + 1) / cuts) - m0;
      int found = 0;
      for (int i = warp * per + lane; i < (warp + 1) * per; i += 32)
        found += __popc(__ballot_sync(0xffffffffu, i < p.pairs && lid[min(i, p.pairs - 1)] == (unsigned)e));
      if (lane == 0) seen[warp] = found;
      __syncthreads();
      int at = (int)__reduce_add_sync(0xffffffffu, lane < warp ? seen[lane] : 0) - m0;
      if (found > 0)
        for (int i = warp * per + lane; i < (warp + 1) * per; i += 32) {
          const bool is = i < p.pairs && lid[min(i, p.pairs - 1)] == (unsigned)e;
          const unsigned m = __ballot_sync(0xffffffffu, is);
          const int k = at + __popc(m & ((1u << lane) - 1));
          if (is && k >= 0 && k < nx) list[k] = i;
          at += __popc(m);
        }
    }
    __syncthreads();
    const int* mine = list;
    {
      const auto row = [&](int r) {
        return p.in + (GATED ? mine[r] / p.topk : (int64_t)(r & 1) * p.pairs + mine[r >> 1]) * p.in_stride;
      };
      const auto emit = [&](int tile, const float (&acc)[2][NT][4]) {
#pragma unroll
        for (int r = 0; r < (GATED ? 2 : 4); ++r) {
          const int n = (ta + tile) * (GATED ? 16 : 32) + r * 8 + g;
          if (n >= (GATED ? p.w.n / 2 : p.w.n)) continue;
          const __nv_bfloat16* b = p.bias == nullptr ? nullptr : p.bias + (int64_t)e * p.w.n + n;
          const float b0 = b == nullptr ? 0.f : __bfloat162float(b[0]);
          const float b1 = !GATED || b == nullptr ? 0.f : __bfloat162float(b[p.w.n / 2]);
#pragma unroll
          for (int q = 0; q < NT; ++q) {
            if constexpr (GATED) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const int m = q * 8 + 2 * t + c;
                if (m >= nx) continue;
                __nv_bfloat16* a = p.a + (int64_t)mine[m] * p.a_stride + n;
                w4_act_parts(w4_gated_act(acc[r][q][c] * kW4Unit + b0, acc[r][q][2 + c] * kW4Unit + b1, p.act), a[0],
                             a[(int64_t)p.pairs * p.a_stride]);
              }
            } else {
              const int m = q * 4 + t;
              const float(&v)[4] = acc[r >> 1][q];
              if (m < nx) p.y[(int64_t)mine[m] * p.w.n + n] = (v[2 * (r & 1)] + v[2 * (r & 1) + 1]) * kW4Unit + b0;
            }
          }
        }
      };
      runs.template run<false>(p.w, (int64_t)e * p.w.tiles + ta, nt, 0, p.w.kc, xs, pitch, nx * columns_of(GATED), row, emit);
    }
    pos += nt;
  }
}

// out[t] = sum over a token's choices, in their order, of weight * y; four columns a thread. A pair's row of y is its
// number, or its place[].
__global__ void __launch_bounds__(128) w4_combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ place,
                                                         const float* __restrict__ weights,
                                                         const int32_t* __restrict__ ids, int E, int e0, int topk, int H,
                                                         __nv_bfloat16* __restrict__ out) {
  pdl_wait();
  pdl_launch();
  const int64_t t = blockIdx.x;
  const int c = (blockIdx.y * 128 + threadIdx.x) * 4;
  if (c >= H) return;
  float v[4] = {};
  for (int j = 0; j < topk; ++j) {
    const int64_t p = t * topk + j;
    if (local_expert(ids[p], e0) >= (unsigned)E) continue;
    const float w = weights[p];
    const float* from = y + (place == nullptr ? p : (int64_t)place[p]) * H + c;
    if (H % 4 == 0) {
      const float4 f = *reinterpret_cast<const float4*>(from);
      v[0] += w * f.x, v[1] += w * f.y, v[2] += w * f.z, v[3] += w * f.w;
    } else {
      for (int i = 0; i < 4 && c + i < H; ++i) v[i] += w * from[i];
    }
  }
  if (H % 4 == 0) {
    *reinterpret_cast<uint2*>(out + t * H + c) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
  } else {
    for (int i = 0; i < 4 && c + i < H; ++i) out[t * H + c + i] = __float2bfloat16(v[i]);
  }
}

// 3 if not even one token's inputs fit beside the rings and lists; `launch` false: only says so
template <int NT, int G, bool Z, bool F, bool GATED>
int launch_experts(ExpertArgs p, bool launch, cudaStream_t s) {
  constexpr auto kernel = w4_experts_kernel<NT, G, Z, F, GATED>;
  constexpr int kRun = w4_run_bytes<NT, G, Z>();
  const int pitch = w4_pitch(p.w.kc * 128) * columns_of(GATED);  // of a pair's rows
  p.rows = std::min(NT * 8 / columns_of(GATED), (kSmemMax - kRun - prelude_bytes(p.E, p.pairs, 1)) / pitch);
  if (p.rows < 1) return 3;
  const int64_t most = (int64_t)(std::min(p.E, p.pairs) + p.pairs / p.rows) * p.w.tiles;
  if (most * 2 >= (1ll << 31)) return 3;
  if (!launch) return 0;
  if (msgl_set_smem<kernel>(kSmemMax) != cudaSuccess) return 4;
  const int smem = kRun + prelude_bytes(p.E, p.pairs, p.rows) + p.rows * pitch;
  const int grid = (int)std::min<int64_t>(msgl_num_sms(), most);
  return w4_launch(kernel, dim3(grid), dim3(w4_threads<NT>()), smem, s, 1, p) == cudaSuccess ? 0 : 4;
}

// One product of experts out of `total`. Columns per pass: 8 while an expert has at most 4 on average (it then rarely has
// more than 8), else 16; a second pass reads the expert's weights again, mostly from L2. 128 experts of 2048 x 768, both
// products with one column a pair: at 4 pairs 77 us with columns of 8 and 81 with 16, at 8 pairs 112 and 100.
template <bool GATED>
int experts_product(const ExpertArgs& p, const MsglW4* w, int total, bool launch, cudaStream_t s) {
  return w4_dispatch(w, [&](auto g, auto z, auto f) {
    return p.pairs * columns_of(GATED) <= 4ll * total ? launch_experts<1, g(), z(), f(), GATED>(p, launch, s)
                              : launch_experts<2, g(), z(), f(), GATED>(p, launch, s);
  });
}

// Pairs of a tile. Up to 64 two sets of accumulators fit into tensor memory beside two stages of A, so that a tile's
// results leave while the next one is multiplied; 128 fit once, and convert the weights half as often. 128 experts of
// 2048 x 768, 8 a token, 64 and 128 a tile: 512 tokens (32 pairs an expert) 181 and 196 us, 1024 tokens 271 and 254, 2048
// tokens 435 and 401, 16384 tokens 3135 and 2656. (80 and 96 lie between.)
constexpr int kTileFew = 64, kTileMany = kGwMaxGather;
inline int tile_tokens(int64_t pairs, int64_t total) { return pairs <= 40 * total ? kTileFew : kTileMany; }

// Sorts the pairs by expert (in any order within one: a pair's result does not depend on its place) and cuts
// every expert's into equal tiles. One CTA.
__global__ void __launch_bounds__(1024) w4_plan_kernel(const int32_t* __restrict__ ids, int pairs, int E, int e0,
                                                       int32_t* __restrict__ sorted, int32_t* __restrict__ place,
                                                       int4* __restrict__ work,
                                                       int32_t* __restrict__ count, int tile) {
  __shared__ int cnt[kMoeMaxExperts], at[kMoeMaxExperts], sums[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch();
  cnt[tid] = 0;
  __syncthreads();
  for (int i = tid; i < pairs; i += 1024) {
    const unsigned e = local_expert(ids[i], e0);
    if (e < (unsigned)E) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  // running sums of the pairs and tiles over the experts, one a thread
  const int c = cnt[tid], tiles = (c + tile - 1) / tile;
  int a = c, b = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += x, b += y;
  }
  if (lane == 31) sums[0][warp] = a, sums[1][warp] = b;
  __syncthreads();
  if (warp == 0) {
    int x = sums[0][lane], y = sums[1][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) x += u, y += v;
    }
    sums[0][lane] = x, sums[1][lane] = y;
    if (lane == 31) *count = y;
  }
  __syncthreads();
  const int start = a - c + (warp > 0 ? sums[0][warp - 1] : 0), first = b - tiles + (warp > 0 ? sums[1][warp - 1] : 0);
  at[tid] = start;
  for (int i = 0; i < tiles; ++i) {
    const int from = (int)((int64_t)c * i / tiles), to = (int)((int64_t)c * (i + 1) / tiles);
    work[first + i] = make_int4(tid, start + from, to - from, 0);
  }
  __syncthreads();
  for (int i = tid; i < pairs; i += 1024) {
    const unsigned e = local_expert(ids[i], e0);
    if (e < (unsigned)E) {
      const int to = atomicAdd(&at[e], 1);
      sorted[to] = i;
      place[i] = to;
    }
  }
}

// scratch of a call: activated rows, results of the pairs, and for many tokens the sorted pairs and tiles
struct Scratch {
  int64_t a, y, sorted, place, work, count, bytes;
};
Scratch scratch_of(int64_t pairs, int E, const MsglW4* w2) {
  const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  Scratch s;
  s.a = 0;
  s.y = up((pairs <= kMoeMaxPairs ? 2 : 1) * pairs * w2->kc * 128 * 2);  // (the streaming product's in two parts)
  s.sorted = s.y + up(pairs * w2->n * 4);
  s.place = s.sorted + up(pairs * 4);
  s.work = s.place + up(pairs * 4);
  s.count = s.work + up((E + pairs / kTileFew) * 16);
  s.bytes = s.count + 256;
  return s;
}

// Pairs per expert up to which the streaming product is taken. 128 experts of 2048 x 768, streaming and on the tensor
// core: at 12 a layer takes 140 and 146 us, at 14 151 and 153, at 16 163 and 156; 32 experts of 2880 x 2880, groups of 32
// with zero points: at 12.5 both 198, at 16 231 and 205. Where only a share of the experts is here, pairs and experts of
// all ranks count: 8 of 64 experts of 2880 x 2880 at 32 tokens, 8 a token, 38 us streaming and 74 on the tensor core.
constexpr int kStreamPairs = 12;

int experts_tiles(const void* x, int64_t x_stride, int pairs, int topk, const MsglW4* w1, const MsglW4* w2, int E, int e0,
                  int total, const int32_t* ids, const void* b1, const void* b2, int act, uint8_t* ws, const Scratch& sc,
                  cudaStream_t s) {
  int32_t *sorted = (int32_t*)(ws + sc.sorted), *count = (int32_t*)(ws + sc.count);
  int4* work = (int4*)(ws + sc.work);
  const int tile = tile_tokens(pairs, total);
  if (w4_launch(w4_plan_kernel, dim3(1), dim3(1024), 0, s, 1, ids, pairs, E, e0, sorted, (int32_t*)(ws + sc.place), work,
                  count, tile) != cudaSuccess)
    return 4;
  W4GemmArgs p = {};
  p.bn = std::min(tile, (pairs + 15) / 16 * 16);
  p.splits = 1;
  p.count = count, p.work = work, p.sorted = sorted;
  p.topk = topk, p.act = act;
  const int64_t tiles = std::min<int64_t>(E + pairs / tile, pairs);
  W4GemmArgs q = p;
  p.w = w4_tensor(w1);
  p.group = w1->group, p.zeros = w1->zeros, p.fp16 = w1->fp16;
  p.in = (const __nv_bfloat16*)x, p.in_stride = x_stride;
  p.bias = (const __nv_bfloat16*)b1;
  p.out = ws + sc.a, p.out_stride = w2->kc * 128;
  p.n_tiles = (w1->tiles + 7) / 8;
  q.w = w4_tensor(w2);
  q.group = w2->group, q.zeros = w2->zeros, q.fp16 = w2->fp16;
  q.in = (const __nv_bfloat16*)(ws + sc.a), q.in_stride = w2->kc * 128;
  q.M = pairs;
  q.bias = (const __nv_bfloat16*)b2;
  q.out = ws + sc.y, q.out_stride = w2->n;
  q.n_tiles = (w2->tiles + 7) / 8;
  const int64_t most = tiles * std::max(p.n_tiles, q.n_tiles);
  if (most >= (1ll << 31)) return 3;
  const int sms = msgl_num_sms();
  const int rc = w4_gemm_launch<kW4GateUp, 2, false>(p, (int)std::min<int64_t>(sms, tiles * p.n_tiles), s);
  return rc != 0 ? rc : w4_gemm_launch<kW4Down, 2, false>(q, (int)std::min<int64_t>(sms, tiles * q.n_tiles), s);
}

}  // namespace

extern "C" int64_t msgl_w4_experts_workspace(int T, int topk, int E, const MsglW4* w1, const MsglW4* w2) {
  return scratch_of((int64_t)T * topk, E, w2).bytes;
}

extern "C" int msgl_w4_experts(void* out, const void* x, int64_t x_stride, int T, int topk, const MsglW4* w1,
                               const MsglW4* w2, int E, int e0, int total, const float* weights, const int32_t* ids,
                               const void* b1, const void* b2, int act, void* workspace, int* launches,
                               cudaStream_t s) {
  *launches = w4_launched = 0;
  if (T == 0) return 0;
  if (E > kMoeMaxExperts) return 3;
  const int pairs = T * topk, a_stride = w2->kc * 128;
  uint8_t* ws = (uint8_t*)workspace;
  const Scratch sc = scratch_of(pairs, E, w2);
  __nv_bfloat16* a = (__nv_bfloat16*)(ws + sc.a);
  const ExpertArgs p1 = {w4_tensor(w1), E, e0, pairs, topk, ids, (const __nv_bfloat16*)x, x_stride, (const __nv_bfloat16*)b1,
                         a, nullptr, a_stride, act, 0};
  const ExpertArgs p2 = {w4_tensor(w2), E, e0, pairs, topk, ids, a, a_stride, (const __nv_bfloat16*)b2, nullptr,
                         (float*)(ws + sc.y), 0, 0, 0};
  // (experts of some 20,000 inputs and more may not fit the streaming products)
  const bool stream = pairs <= (int64_t)kStreamPairs * total && pairs <= kMoeMaxPairs &&
                      experts_product<true>(p1, w1, total, false, s) == 0 && experts_product<false>(p2, w2, total, false, s) == 0;
  int rc;
  if (stream) {
    rc = experts_product<true>(p1, w1, total, true, s);
    if (rc == 0) rc = experts_product<false>(p2, w2, total, true, s);
  } else {
    rc = experts_tiles(x, x_stride, pairs, topk, w1, w2, E, e0, total, ids, b1, b2, act, ws, sc, s);
  }
  if (rc == 0 &&
      w4_launch(w4_combine_kernel, dim3(T, (w2->n + 511) / 512), dim3(128), 0, s, 1, (const float*)(ws + sc.y),
                stream ? (const int32_t*)nullptr : (const int32_t*)(ws + sc.place), weights, ids, E, e0, topk, w2->n,
                (__nv_bfloat16*)out) != cudaSuccess)
    rc = 4;
  *launches = w4_launched;
  return rc;
}

MSGL_ERROR_ACCESSOR(msgl_err_w4_moe)
