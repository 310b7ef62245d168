// Ragged causal attention over the paged 8-bit cache.
//
// o_i = sum_j w_ij s^v_j c^v_j / sum_j w_ij with w_ij = exp(scale s^k_j q_i . c^k_j) over the keys that query i sees.
//
// One warp per (token, head): its lanes hold the head dims, every key is one dot product over the warp.
#include <algorithm>

#include "api.h"
#include "common.cuh"
#include "kv8.cuh"

using namespace msgl;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// A request's queries and keys, with what is outside its tables taken out (and recorded).
struct Kv8Req {
  int q0, n, L, row;
};
__device__ __forceinline__ Kv8Req kv8_request(const Kv8Attn& p, int b) {
  Kv8Req r;
  const int a = p.cu_q[b], e = p.cu_q[b + 1];
  r.q0 = min(max(a, 0), p.total_q);
  r.n = min(max(e, r.q0), p.total_q) - r.q0;
  r.L = p.kv_lens[b];
  r.row = p.rows[b];
  const bool ok = r.q0 == a && r.q0 + r.n == e && r.L >= 0 && r.L <= p.pt_width && (r.L == 0 || (r.row >= 0 && r.row < p.pt_rows));
  if (!ok) {
    report_error(kErrBounds, kBcAttnRow);
    r.L = 0;
  }
  return r;
}
// First slot of the page that holds position `pos` (a multiple of the page), or -1.
__device__ __forceinline__ int kv8_page(const Kv8Attn& p, int row, int pos) {
  const int slot = p.page_table[(int64_t)row * p.pt_stride + pos];
  if (slot < 0 || slot > p.num_slots - p.page || slot % p.page != 0) {
    report_error(kErrBounds, kBcAttnSlot);
    return -1;
  }
  return slot;
}

template <int HD, bool FP8>
__global__ void __launch_bounds__(128) kv8_attention_simple(Kv8Attn p) {
  pdl_wait();
  pdl_launch();
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= (int64_t)p.total_q * p.nq) return;
  const int t = (int)(w / p.nq), head = (int)(w % p.nq), h = head / (p.nq / p.nkv);
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.o) + w * HD;
  constexpr int E = HD / 32;
  int lo = 0, hi = p.num_reqs;  // the request of token t: the last one that starts at or before it and has queries
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (p.cu_q[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= p.num_reqs) {
    if (p.zero_tail)
      for (int e = 0; e < E; ++e) o[lane * E + e] = __float2bfloat16(0.f);
    return;
  }
  const Kv8Req r = kv8_request(p, lo);
  const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q) + t * p.q_row + head * p.q_head;
  float qv[E], acc[E];
  for (int e = 0; e < E; ++e) qv[e] = __bfloat162float(q[lane * E + e]), acc[e] = 0.f;
  const int pos = r.L - r.n + (t - r.q0), end = r.L == 0 ? 0 : pos + 1;
  float m = -INFINITY, l = 0.f;
  int page = -1;
  for (int j = p.window > 0 ? max(0, pos - p.window + 1) : 0, fresh = 1; j < end; ++j, fresh = 0) {
    if (fresh || j % p.page == 0) page = kv8_page(p, r.row, j - j % p.page);
    float k[E], v[E], ks = 0.f, vs = 0.f;
    for (int e = 0; e < E; ++e) k[e] = v[e] = 0.f;
    if (page >= 0) {
      const int64_t at = (int64_t)h * p.num_slots + page + j % p.page;
      ks = p.sk[at], vs = p.sv[at];
      for (int e = 0; e < E; e += 2) {
        const float2 a = kv8_decode2<FP8>(reinterpret_cast<const uint16_t*>(p.ck)[(at * HD + lane * E + e) / 2]);
        const float2 b = kv8_decode2<FP8>(reinterpret_cast<const uint16_t*>(p.cv)[(at * HD + lane * E + e) / 2]);
        k[e] = a.x, k[e + 1] = a.y, v[e] = b.x, v[e + 1] = b.y;
      }
    }
    float s = 0.f;
    for (int e = 0; e < E; ++e) s += qv[e] * k[e];
    s = warp_sum(s) * ks * p.scale * kLog2e;
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn, f = exp2f(m - base), x = exp2f(s - base);
    l = l * f + x;
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + x * vs * v[e];
    m = mn;
  }
  float f = 1.f;
  if (p.sinks != nullptr && l > 0.f) {
    const float sink = p.sinks[head] * kLog2e, mn = fmaxf(m, sink);
    f = exp2f(m - mn);
    l = l * f + exp2f(sink - mn);
  }
  const float inv = l == 0.f ? 0.f : f / l;
  for (int e = 0; e < E; ++e) o[lane * E + e] = __float2bfloat16(acc[e] * inv);
}

}  // namespace

extern "C" int msgl_kv8_attention(const Kv8Attn* p, int hd, int fp8, int max_q_len, int* launches, cudaStream_t s) {
  (void)max_q_len;
  const int64_t blocks = ((int64_t)p->total_q * p->nq + 3) / 4;
  if ((hd != 64 && hd != 128) || blocks > INT32_MAX) return 3;
  auto* f = hd == 64 ? (fp8 ? kv8_attention_simple<64, true> : kv8_attention_simple<64, false>)
                     : (fp8 ? kv8_attention_simple<128, true> : kv8_attention_simple<128, false>);
  *launches = 1;
  return msgl_launch(f, dim3((unsigned)blocks), dim3(128), 0, s, 1, *p) == cudaSuccess ? 0 : 4;
}

MSGL_ERROR_ACCESSOR(msgl_err_kv8_attn)
