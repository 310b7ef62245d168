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
// lowest), so every v is finite and the order is total: that of 64-bit arithmetic.
//
// One warp per token. The choice is made in fp32, with a bound on its errors: where two values that the
// choice depends on are nearer than that (a few rows in a thousand), the candidates or the groups are looked at
// again in 64 bits; without a bias the logits themselves decide and nothing is near. 16384 tokens x 256
// experts, 8 of them, fp32 logits: 13 us softmax (490 warp instructions a token), 26 us with sigmoid scores, bias and
// groups (900), against 2.8 us for the bytes; every row in 64 bits took 65 us. What bounds both is waiting: with the 24
// and 16 warps an SM that the registers leave, 65% and 55% of the issue slots are used, and the rest goes to chains of
// dependent instructions, to shuffles and shared memory, and to the chosen logits' second read.
//
// The weights: an expf, over the sum of the row's fast exponentials (softmax without renormalising) or of the chosen
// scores. The exponent's rounding counts |logit - largest| times 2^-24: down to scores of e^-32 of the largest a weight is
// off by 2^-18 of its value at most, as a rule by 2^-23.
//
// Top k: the (k + 1)-th largest of the lanes' maxima (a sort of 32 keys across the warp) bounds the
// (k + 1)-th largest value from below; the few values at or above it are gathered, a lane each, and ranked by
// comparing each with each. Rows with more than 32 of them (many equal values) pick one after another.
#include <cfloat>

#include "api.h"
#include "common.cuh"

using namespace msgl;

namespace {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxE = 512;
// CTAs per SM. At 6 (80 registers) the forms without groups spill 8 to 32 bytes for 128 and 256 experts, 140 between and
// some 200 above them; with groups, at 4 (128 registers), only those above 256 experts do (about 110 bytes).
__host__ __device__ constexpr int route_ctas(bool groups) { return groups ? 4 : 6; }

struct RouteArgs {
  const void* logits;
  int64_t stride;
  const float* bias;
  int n_tok, E, topk, sigmoid, groups, kept, top2, renorm;
  int per, lanes, log_lanes;  // experts of a group, lanes of a group and their logarithm
  float scale;
  float* weights;
  int32_t* ids;
};

template <typename T>
__device__ __forceinline__ float logit_of(const T* p);
template <>
__device__ __forceinline__ float logit_of<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float logit_of<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// (+ 0.f: -0 and 0 are equal, and so are their keys)
// fmaxf takes the other operand of a NaN
__device__ __forceinline__ float clean_logit(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX) + 0.f; }
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

// One token in 64 bits, with 2 E doubles of scratch.
template <typename T>
__device__ __noinline__ void route_exact(const RouteArgs& a, const T* row, int t, double* p) {
  const int lane = threadIdx.x & 31, E = a.E, topk = a.topk, groups = a.groups;
  double* v = p + E;  // what the choice goes by
  const bool by_logit = a.bias == nullptr;

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
    if (a.sigmoid) s = 1.0 / (1.0 + exp(-x));
    else s = mx == -INFINITY ? 0.0 : exp(x - mx);
    v[e] = by_logit ? fmax(x, -(double)FLT_MAX * 2) : (double)clean_bias(a.bias[e]);
    p[e] = s;
    sum += s;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  for (int e = lane; e < E; e += 32) {
    if (!a.sigmoid) p[e] = sum > 0.0 ? p[e] / sum : 0.0;
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
      double c = -INFINITY, d = -INFINITY;
      for (int j = 0; j < per; ++j) {
        const double x = (by_logit && a.top2) ? p[g * per + j] : v[g * per + j];
        if (x > c) { d = c; c = x; } else if (x > d) d = x;
      }
      rank[i] = a.top2 ? c + d : c;
    }
    unsigned keep = 0;  // bit i: this lane's group lane + 32 i stays
    for (int n = 0; n < a.kept; ++n) {
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
      a.ids[(int64_t)t * topk + n] = bi;
      v[bi] = -INFINITY;
    }
    __syncwarp();
  }
  if (lane < topk) {
    const double w = p[a.ids[(int64_t)t * topk + lane]];
    a.weights[(int64_t)t * topk + lane] = (float)((a.renorm ? (total > 0.0 ? w / total : 0.0) : w) * (double)a.scale);
  }
}

// unsigned keys in the order of the floats; 0 is below all of them
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ float sigmoid_of(float x) { return __fdividef(1.f, 1.f + expf(-x)); }

// e^x on the MUFU unit, for the choice: off by 2^-22 and the rounding of x log2 e, which |x| <= 16 makes 2^-20 of the
// value at most and a smaller part of the largest score where |x| is larger
__device__ __forceinline__ float exp_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

// the lane's place among the first n lanes' keys, largest first, equal ones by lane; lanes from n on have 0
__device__ __forceinline__ int place_of(uint32_t key, int n) {
  int r = __popc(__match_any_sync(0xffffffffu, key) & ((1u << (threadIdx.x & 31)) - 1));
  for (int j = 0; j < n; j += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) r += __shfl_sync(0xffffffffu, key, j + i) > key;
  return r;
}

// e^(l - mx) over a row, and an expert's score + bias, in 64 bits
template <typename T>
__device__ __noinline__ double sum_exact(const T* row, int E, float mx) {
  double sum = 0.0;
  if (mx != -INFINITY)
    for (int e = threadIdx.x & 31; e < E; e += 32) sum += exp((double)clean_logit(logit_of(row + e)) - mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
template <typename T>
__device__ __noinline__ double value_exact(const RouteArgs& a, const T* row, int e, float mx, double sum) {
  const double l = clean_logit(logit_of(row + e));
  const double p = a.sigmoid ? 1.0 / (1.0 + exp(-l)) : sum > 0.0 ? exp(l - mx) / sum : 0.0;
  return a.bias == nullptr ? p : p + clean_bias(a.bias[e]);
}

// The groups that stay (bit g << log_lanes), from scores in 64 bits; v: E doubles of scratch.
template <typename T>
__device__ __noinline__ unsigned groups_exact(const RouteArgs& a, const T* row, float mx, double* v) {
  const int lane = threadIdx.x & 31, L = a.lanes, g = lane >> a.log_lanes;
  const double sum = a.sigmoid ? 0.0 : sum_exact(row, a.E, mx);
  __syncwarp();
  for (int e = lane; e < a.E; e += 32) v[e] = value_exact(a, row, e, mx, sum);
  __syncwarp();
  double c = -INFINITY, d = -INFINITY;
  if (g < a.groups)
    for (int j = lane & (L - 1); j < a.per; j += L) {
      const double o = v[g * a.per + j];
      d = fmax(d, fmin(c, o));
      c = fmax(c, o);
    }
  for (int o = 1; o < L; o <<= 1) {
    const double c2 = __shfl_xor_sync(0xffffffffu, c, o), d2 = __shfl_xor_sync(0xffffffffu, d, o);
    d = fmax(fmax(d, d2), fmin(c, c2));
    c = fmax(c, c2);
  }
  const double rank = a.top2 ? c + d : c;
  int place = 0;
  for (int j = 0; j < a.groups; ++j) {
    const double o = __shfl_sync(0xffffffffu, rank, j * L);
    place += o > rank || (o == rank && j < g);
  }
  __syncwarp();
  return __ballot_sync(0xffffffffu, place < a.kept && g < a.groups);
}

// what the lane's experts keep over the tokens: their biases, and with groups (e = lane + 32 i, g its group) the place
// of their values in the scratch, e + g L, and the first of the group's lanes, g L
template <int PER, bool GROUPS>
struct LaneExperts {
  float bias[PER];
  int at[GROUPS ? PER : 1], first[GROUPS ? PER : 1];
};

// One token. x: the lane's logits, of experts lane + 32 i; FULL: there are exactly 32 PER.
template <typename T, int PER, bool GROUPS, bool FULL>
__device__ __forceinline__ void route_token(const RouteArgs& a, const LaneExperts<PER, GROUPS>& le, const T* row, int t, double* scratch,
                                            float (&x)[PER]) {
  const int lane = threadIdx.x & 31, E = FULL ? 32 * PER : a.E;
  const bool by_logit = a.bias == nullptr, sums = GROUPS && a.top2;
  uint32_t key[PER];
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool in = FULL || lane + 32 * i < E;
    x[i] = in ? clean_logit(x[i]) : -INFINITY;
    key[i] = in ? key_of(x[i]) : 0u;
    mx = fmaxf(mx, x[i]);
  }
  float inv = 0.f, top_p = 1.f;  // softmax: 1 / the sum of the exponentials; no score is above top_p
  if (!a.sigmoid) {
    mx = warp_max(mx);
    if (!by_logit || sums || !a.renorm) {
      float sum = 0.f;
      const float m = mx == -INFINITY ? 0.f : mx;  // then every exponential is zero
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += exp_fast(x[i] - m);
      sum = warp_sum(sum);
      inv = top_p = sum > 0.f ? 1.f / sum : 0.f;
    }
  }
  // Errors: a sigmoid is off by 2^-20 and a few roundings (2^-19 of the largest possible, 1), a softmax score by
  // the roundings of its sum too (32 at most: 2^-18 of the largest, top_p), p + bias by its own rounding too. Values
  // further apart than near() of the larger magnitude are in order, and so is whatever lies beyond them: a value that
  // is far away (a bias that masks an expert) has a larger error, but not one that brings it back.
  const float err = (a.sigmoid ? 0x1p-19f : 0x1p-18f) * top_p;
  const auto near = [err](float v) { return 2.f * err + 0x1p-22f * fabsf(v); };
  if (!by_logit || sums) {
    if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = __fdividef(1.f, 1.f + exp_fast(-x[i]));
    } else {
      const float m = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = exp_fast(x[i] - m) * inv;
    }
    if (!by_logit) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (FULL || lane + 32 * i < E) {
          x[i] += le.bias[i];
          key[i] = key_of(x[i]);
        }
    }
  }

  const bool exact = GROUPS && a.groups > 32;  // more groups than lanes
  if (GROUPS && !exact) {
    // L lanes share a group: each keeps its two largest, and they merge. The groups lie L words further apart
    // than their size, so that groups of 32 do not meet in the banks.
    const int per = a.per, L = a.lanes;
    uint32_t* gk = reinterpret_cast<uint32_t*>(scratch);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (FULL || lane + 32 * i < E) gk[le.at[i]] = by_logit && sums ? key_of(x[i]) : key[i];
    }
    __syncwarp();
    const int g = lane >> a.log_lanes, q = lane & (L - 1);
    uint32_t c = 0, d = 0;
    if (g < a.groups)
#pragma unroll 4
      for (int j = q; j < per; j += L) {
        const uint32_t o = gk[g * (per + L) + j];
        d = max(d, min(c, o));
        c = max(c, o);
      }
    for (int o = 1; o < L; o <<= 1) {
      const uint32_t c2 = __shfl_xor_sync(0xffffffffu, c, o), d2 = __shfl_xor_sync(0xffffffffu, d, o);
      d = max(max(d, d2), min(c, c2));
      c = max(c, c2);
    }
    // every lane of a group has its rank (a sum is held to the finite values: beyond them 64 bits decide)
    const uint32_t rank = g >= a.groups ? 0u : a.top2 ? key_of(fmaxf(fminf(of_key(c) + of_key(d), FLT_MAX), -FLT_MAX)) : c;
    int place = 0;
    for (int j = 0; j < a.groups; ++j) {
      const uint32_t o = __shfl_sync(0xffffffffu, rank, j * L);
      place += o > rank || (o == rank && j < g);
    }
    unsigned stay = __ballot_sync(0xffffffffu, place < a.kept && g < a.groups);
    if (a.kept < a.groups && (sums || !by_logit)) {
      // the last group that stays and the first that does not
      const int in = __ffs(__ballot_sync(0xffffffffu, place == a.kept - 1 && g < a.groups)) - 1;
      const int out = __ffs(__ballot_sync(0xffffffffu, place == a.kept && g < a.groups)) - 1;
      const float u = of_key(__shfl_sync(0xffffffffu, rank, in)), w = of_key(__shfl_sync(0xffffffffu, rank, out));
      // values of opposite signs leave a sum smaller than its errors: the most that any group's two cancel
      // (lanes without a group have keys of NaN, which fmaxf drops)
      float gone = 0.f;
      if (a.top2) gone = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fminf(of_key(c), -of_key(d)), 0.f))));
      if (!(u - w > 2.f * near(fmaxf(fabsf(u), fabsf(w))) + 0x1p-21f * gone)) stay = groups_exact(a, row, mx, scratch);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (!((stay >> le.first[i]) & 1)) key[i] = 0;
    __syncwarp();
  }
  if (exact) {
    route_exact<T>(a, row, t, scratch);
    return;
  }

  // the (k + 1)-th largest of the lanes' maxima
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) top = max(top, key[i]);
  uint32_t sorted = top;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, sorted, o);
      const bool larger = ((lane & size) == 0) == ((lane & o) == 0);  // descending in the end
      sorted = larger ? max(sorted, other) : min(sorted, other);
    }
  uint32_t floor_key = a.topk < 32 ? max(__shfl_sync(0xffffffffu, sorted, a.topk & 31), 1u) : 1u;
  // what may be one of the k + 1 largest in truth
  if (!by_logit && floor_key > 1u) floor_key = max(key_of(of_key(floor_key) - near(of_key(floor_key))), 1u);
  uint2* cand = reinterpret_cast<uint2*>(scratch);  // {key, expert}, room for all of them
  int n = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool in = key[i] >= floor_key;
    const unsigned m = __ballot_sync(0xffffffffu, in);
    if (in) cand[n + __popc(m & ((1u << lane) - 1))] = make_uint2(key[i], lane + 32 * i);
    n += __popc(m);
  }
  __syncwarp();
  // chosen: lane r has the r-th
  uint32_t ckey = 0;
  int cid = 0;
  if (n <= 32) {
    const uint2 mine = lane < n ? cand[lane] : make_uint2(0, 0);
    const int r = place_of(mine.x, n);
    __syncwarp();
    if (lane < n) cand[r] = mine;
    __syncwarp();
    if (lane < n) ckey = cand[lane].x, cid = (int)cand[lane].y;
  } else {
    for (int k = 0; k <= a.topk && k < 32; ++k) {
      uint32_t b = 0;
      int bi = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (key[i] > b) b = key[i], bi = i;
      const uint32_t m = __reduce_max_sync(0xffffffffu, b);
      const uint32_t e = __reduce_min_sync(0xffffffffu, b == m ? (uint32_t)(lane + 32 * bi) : 0xffffffffu);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if ((uint32_t)(lane + 32 * i) == e) key[i] = 0;
      if (lane == k) ckey = m, cid = (int)e;
    }
  }
  if (!by_logit) {
    const float v = of_key(ckey), next = of_key(__shfl_down_sync(0xffffffffu, ckey, 1));
    // the last candidate has nothing behind it; with 32 chosen the 33rd is not known
    const bool behind = lane < a.topk && lane + 1 < min(n, 32);
    if (__any_sync(0xffffffffu, behind && !(v - next > near(fmaxf(fabsf(v), fabsf(next))))) || (a.topk == 32 && n > 32)) {
      if (n > 32) {
        __syncwarp();
        route_exact<T>(a, row, t, scratch);
        return;
      }
      // the candidates again in 64 bits, and their order
      const double sum = a.sigmoid ? 0.0 : sum_exact(row, E, mx);
      const double w = lane < n ? value_exact(a, row, cid, mx, sum) : -INFINITY;
      int r = 0;
      for (int k = 0; k < n; ++k) {
        const double o = __shfl_sync(0xffffffffu, w, k);
        const int e = __shfl_sync(0xffffffffu, cid, k);
        r += o > w || (o == w && e < cid);
      }
      if (lane < n) cand[r] = make_uint2(ckey, cid);
      __syncwarp();
      if (lane < n) cid = (int)cand[lane].y;
    }
  }
  float p = 0.f;
  if (lane < a.topk) {
    const float l = clean_logit(logit_of(row + cid));
    p = a.sigmoid ? sigmoid_of(l) : mx == -INFINITY ? 0.f : expf(l - mx) * (inv > 0.f ? inv : 1.f);
  }
  if (a.renorm) {
    const float total = warp_sum(p);
    if (!(total > 0x1p-80f)) {  // scores at the end of fp32's range (or zero)
      __syncwarp();
      route_exact<T>(a, row, t, scratch);
      return;
    }
    p = __fdividef(p, total);
  }
  if (lane < a.topk) {
    a.weights[(int64_t)t * a.topk + lane] = p * a.scale;
    a.ids[(int64_t)t * a.topk + lane] = cid;
  }
}

// PER: experts of a lane. The warps take the tokens in turn; a token's logits are on their way while the one before
// it is done.
template <typename T, int PER, bool GROUPS, bool FULL>
__global__ void __launch_bounds__(kRouteWarps * 32, route_ctas(GROUPS)) route_experts_kernel(const __grid_constant__ RouteArgs a) {
  pdl_wait();
  pdl_launch();
  extern __shared__ double route_sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = FULL ? 32 * PER : a.E;
  double* scratch = route_sm + (size_t)warp * (2 * E + 32);
  const T* base = reinterpret_cast<const T*>(a.logits);
  const int step = gridDim.x * kRouteWarps;
  float next[PER];
  LaneExperts<PER, GROUPS> le;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    le.bias[i] = a.bias != nullptr && e < E ? clean_bias(__ldg(a.bias + e)) : 0.f;
    if constexpr (GROUPS) le.first[i] = e / a.per * a.lanes & 31, le.at[i] = e + e / a.per * a.lanes;
  }
  const auto fetch = [&](int t) {
    const T* row = base + (int64_t)t * a.stride + lane;
#pragma unroll
    for (int i = 0; i < PER; ++i) next[i] = FULL || lane + 32 * i < E ? logit_of(row + 32 * i) : 0.f;
  };
  int t = blockIdx.x * kRouteWarps + warp;
  if (t >= a.n_tok) return;
  fetch(t);
  for (;; t += step) {
    float x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = next[i];
    const bool more = a.n_tok - t > step;  // (t + step may be beyond 31 bits)
    if (more) fetch(t + step);
    route_token<T, PER, GROUPS, FULL>(a, le, base + (int64_t)t * a.stride, t, scratch, x);
    if (!more) return;
    __syncwarp();
  }
}

template <typename T, int PER>
cudaError_t launch_route_per(const RouteArgs& a, cudaStream_t s) {
  const size_t smem = (size_t)kRouteWarps * (2 * a.E + 32) * sizeof(double);
  const int ctas = (a.n_tok - 1) / kRouteWarps + 1, most = msgl_num_sms() * route_ctas(a.groups > 1);
  const dim3 grid(ctas < most ? ctas : most), block(kRouteWarps * 32);
  if (a.E == 32 * PER)
    return a.groups > 1 ? msgl_launch(route_experts_kernel<T, PER, true, true>, grid, block, smem, s, 1, a)
                        : msgl_launch(route_experts_kernel<T, PER, false, true>, grid, block, smem, s, 1, a);
  return a.groups > 1 ? msgl_launch(route_experts_kernel<T, PER, true, false>, grid, block, smem, s, 1, a)
                      : msgl_launch(route_experts_kernel<T, PER, false, false>, grid, block, smem, s, 1, a);
}

template <typename T>
cudaError_t launch_route(const RouteArgs& a, cudaStream_t s) {
  if (a.E <= 32) return launch_route_per<T, 1>(a, s);
  if (a.E <= 64) return launch_route_per<T, 2>(a, s);
  if (a.E <= 128) return launch_route_per<T, 4>(a, s);
  if (a.E <= 256) return launch_route_per<T, 8>(a, s);
  return launch_route_per<T, 16>(a, s);
}

}  // namespace

extern "C" int msgl_route_experts(const void* logits, int is_fp32, int64_t stride, const float* bias, int n_tok, int E,
                                  int topk, int sigmoid, int groups, int kept, int top2, int renorm, float scale,
                                  float* weights, int32_t* ids, cudaStream_t s) {
  if (n_tok == 0) return 0;
  if (E < 1 || E > kRouteMaxE || topk < 1 || topk > 32 || groups < 1 || groups > 256 || E % groups != 0) return 3;
  const int per = E / groups;
  int log_lanes = 5;
  while (log_lanes > 0 && (groups << log_lanes) > 32) --log_lanes;
  const RouteArgs a = {logits, stride, bias, n_tok, E, topk, sigmoid, groups, kept, top2, renorm,
                       per, 1 << log_lanes, log_lanes, scale, weights, ids};
  const cudaError_t e = is_fp32 ? launch_route<float>(a, s) : launch_route<__nv_bfloat16>(a, s);
  return e == cudaSuccess ? 0 : 4;
}
