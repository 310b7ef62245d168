// How attention over the 8-bit cache spreads its work, and how it joins what was cut.
//
// The rows of a request and kv head are its (token, head of the group) pairs, packed: row r is token r / G, head r % G,
// so a key read once serves the whole group. A segment is a tile of R rows and the 64-key blocks that any of them
// sees (at least one, empty or not). It counts as its blocks plus COST units, what starting and ending it takes. All
// segments' units, request by request, head by head, tile by tile, form one row that is cut into P equal runs, one per
// CTA: lengths of any mixture balance without a work list from the host, and a graph replays with new ones. A CTA
// finds its run by a scan over the requests. Whole segments are written out at once; a run has at most one part of a
// segment at its start and one at its end, so there are 2 P slots for parts whatever the lengths, and a second kernel
// joins each cut segment from its first part's header. (Counters that let the last part's CTA do that would have to be
// zeroed by a launch as well, or shared between calls.)
#pragma once
#include "api.h"
#include "kv8.cuh"

namespace msgl {

constexpr int kKv8Block = 64;  // keys per unit
constexpr float kKv8Log2e = 1.4426950408889634f;

// A request's queries and keys, with what is outside its tables taken out (and recorded).
struct Kv8Req {
  int q0, n, L, row;
};
MSGL_DEVICE Kv8Req kv8_request(const Kv8Attn& p, int b) {
  Kv8Req r;
  const int a = p.cu_q[b], e = p.cu_q[b + 1];
  r.L = p.kv_lens[b];
  r.row = p.rows[b];
  r.q0 = min(max(a, 0), p.total_q);
  r.n = min(max(e, r.q0), p.total_q) - r.q0;
  const bool ok = r.q0 == a && r.q0 + r.n == e && (b > 0 || a == 0) && r.L >= 0 && r.L <= p.pt_width && (r.L == 0 || (r.row >= 0 && r.row < p.pt_rows));
  if (!ok) {
    report_error(kErrBounds, kBcAttnRow);
    r.L = 0;
  }
  return r;
}

// Packed row x of a request: its token.
MSGL_DEVICE int kv8_token(const Kv8Attn& p, int x) { return (int)((uint64_t)(uint32_t)x * p.group_mul >> p.group_shift); }

// A page's first slot as the table has it, or -1 if there is no such page (recorded).
MSGL_DEVICE int kv8_checked(const Kv8Attn& p, int slot) {
  if (slot < 0 || slot > p.num_slots - p.page || slot % p.page != 0) {
    report_error(kErrBounds, kBcAttnSlot);
    return -1;
  }
  return slot;
}

// Tile t of a request: rows [r0, r0 + nr), the positions of the first and the last of them, the keys [lo, kend)
// that any of them sees and the blocks [blk0, blk0 + nblk) that hold those.
struct Kv8Tile {
  int r0, nr, pos0, pos1, lo, kend, blk0, nblk;
};
MSGL_DEVICE Kv8Tile kv8_tile(const Kv8Attn& p, const Kv8Req& r, int G, int R, int t) {
  Kv8Tile k;
  k.r0 = t * R;
  k.nr = min(R, r.n * G - k.r0);
  k.pos0 = r.L - r.n + kv8_token(p, k.r0);
  k.pos1 = r.L - r.n + kv8_token(p, k.r0 + k.nr - 1);
  k.kend = max(0, k.pos1 + 1);
  k.lo = p.window > 0 ? max(0, max(k.pos0, -1) - p.window + 1) : 0;
  k.blk0 = k.lo / kKv8Block;
  k.nblk = max(1, (k.kend > 0 ? (k.kend - 1) / kKv8Block + 1 : 0) - k.blk0);
  return k;
}
MSGL_DEVICE int kv8_tiles(const Kv8Req& r, int G, int R) { return (r.n * G - 1 + R) / R; }  // (r.n * G + 256 fits: rows are less than 2^30)

// A CTA's run of units [u0, u1), and the segment that u0 is in: tile t of head h of request b, from unit s0 on.
struct Kv8Plan {
  int64_t total, u0, u1, s0;
  int ctas, b, h, t;
  Kv8Req r;
};
// the CTA whose run holds unit u: runs are [total c / P, total (c + 1) / P)
MSGL_DEVICE int kv8_cta_of(const Kv8Plan& pl, int64_t u) {
  if (pl.total < (1 << 20)) return (int)(((uint32_t)(u + 1) * pl.ctas - 1) / (uint32_t)pl.total);  // (64-bit divisions are long)
  return (int)(((u + 1) * pl.ctas - 1) / pl.total);
}

// All NT threads of the CTA; `red` holds NT / 32 words. A run has at least `least` units.
template <int COST, int NT>
MSGL_DEVICE void kv8_plan(const Kv8Attn& p, int R, int least, Kv8Plan* pl, int64_t* red) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = p.nq / p.nkv;
  // `per` threads for each request, a power of two: they take its tiles in turn
  int per = 1;
  while (per < 32 && 2 * per * (int64_t)p.num_reqs <= NT) per *= 2;
  const int sub = lane & (per - 1), at_once = NT / per, rounds = max(1, (p.num_reqs + at_once - 1) / at_once);
  int64_t base = 0, v = 0, excl = 0, run0 = 0, run1 = 0;
  int tiles = 0;
  Kv8Req r;
  // one round over the requests, `at_once` at a time: v the units of request (round, tid / per), in its first thread, excl those
  // before it
  auto scan = [&](int c, bool again) {
    const int b = c * at_once + tid / per;
    v = 0;
    tiles = 0;
    if (b < p.num_reqs) {
      r = kv8_request(p, b);
      tiles = kv8_tiles(r, G, R);
#pragma unroll 1
      for (int t = sub; t < tiles; t += per) v += kv8_tile(p, r, G, R, t).nblk + COST;
    }
#pragma unroll 1
    for (int o = per / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    v = sub == 0 ? v * p.nkv : 0;
    int64_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (again) __syncthreads();
    if (lane == 31) red[warp] = incl;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      if (w < warp) before += red[w];
      all += red[w];
    }
    excl = base + before + incl - v;
    base += all;
  };
  auto place = [&](int c) {
    v = __shfl_sync(0xffffffffu, v, lane - sub);
    excl = __shfl_sync(0xffffffffu, excl, lane - sub);
    if (run0 < excl || run0 >= excl + v || run0 >= run1) return;
    // the threads of the request that the run begins in: its head, then its tile, `per` at a time
    const unsigned group = (per == 32 ? 0xffffffffu : (1u << per) - 1) << (lane - sub);
    const int64_t head = v / p.nkv;
    int64_t rem = run0 - excl;
    const int h = v <= UINT32_MAX ? (int)((uint32_t)rem / (uint32_t)head) : (int)(rem / head);
    rem -= h * head;
#pragma unroll 1
    for (int t0 = 0; t0 < tiles; t0 += per) {
      const int t = t0 + sub, units = t < tiles ? kv8_tile(p, r, G, R, t).nblk + COST : 0;
      int64_t incl = units;
#pragma unroll 1
      for (int o = 1; o < per; o <<= 1) {
        const int64_t x = __shfl_up_sync(group, incl, o, per);
        if (sub >= o) incl += x;
      }
      if (rem >= incl - units && rem < incl) {
        pl->b = c * at_once + tid / per;
        pl->r = r;
        pl->h = h;
        pl->t = t;
        pl->s0 = run0 - (rem - (incl - units));
      }
      const int64_t sum = __shfl_sync(group, incl, per - 1, per);
      if (rem < sum) break;
      rem -= sum;
    }
  };
  // All rounds for the total, and, if there are several, once more for the run's place. (One copy of this code, and loops that stay
  // loops: it runs once, and comes out of the L2 cache when it does.)
  const int steps = rounds == 1 ? 1 : 2 * rounds;
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    const int c = step < rounds ? step : step - rounds;
    if (step == rounds) base = 0;
    scan(c, step > 0);
    if (step == rounds - 1) {
      const int64_t total = base;
      int ctas = gridDim.x;
      if (total < (int64_t)ctas * least) ctas = max(1, (int)total / least);
      const int me = blockIdx.x;
      if (me < ctas) {
        const bool small = total < (1 << 20);
        run0 = small ? (uint32_t)total * me / ctas : total * me / ctas;
        run1 = small ? (uint32_t)total * (me + 1) / ctas : total * (me + 1) / ctas;
      }
      if (tid == 0) {
        pl->total = total;
        pl->ctas = ctas;
        pl->u0 = run0;
        pl->u1 = run1;
      }
    }
    if (rounds == 1 || step >= rounds) place(c);
  }
  __syncthreads();
}

// Which of a page's two parts holds the keys' (0 or 1): the tensor maps' base is the lower of the two addresses.
struct Kv8Order {
  int codes, scales;
};

// The copies of one 64-key block, a page at a time: its keys' and values' codes with one instruction, its scales with
// another. Lanes first .. first + pages - 1 hold the pages'
// slots, -1 for a page that is not there: what lies outside the tensors is filled with zeros. (UNROLL: 4 pages at a time are worth 1%
// of a stream of 100000 keys, one at a time, in less code, 2% of prompts on the tensor core.) A page's keys are
// beside its values, codes and scales alike.
template <int HD, int UNROLL>
MSGL_DEVICE void kv8_copy_block(const Kv8Attn& p, const CUtensorMap* tc, const CUtensorMap* ts, uint8_t* codes, float* scales, uint64_t* bar,
                                int h, int slots, int first, int pages) {
  const int page = p.page;
  if (elect_one()) mbar_expect_tx(bar, 2 * page * pages * (HD + 4));
  __syncwarp();
#pragma unroll UNROLL
  for (int i = 0; i < pages; ++i) {
    int slot = __shfl_sync(0xffffffffu, slots, first + i);
    if (slot < 0) slot = p.num_slots;
    if (elect_one()) {
      kv8_load_4d(codes + 2 * i * page * HD, tc, bar, 0, slot, h, 0);
      tma_load_3d(scales + 2 * i * page, ts, bar, slot, h, 0);
    }
    __syncwarp();
  }
}

// Scratch of one call: a header per CTA (of the segment that its run ends in, if cut there and begun in it), and per
// slot the rows' maxima and sums (the logits' log2 domain) and their sums of values.
struct Kv8Part {
  int parts, q0, r0, nr, h, pad[3];  // parts 0: nothing to join
};
struct Kv8Scratch {
  Kv8Part* head;  // [ctas]
  float2* ml;     // [2 ctas][R]
  float* o;       // [2 ctas][R][HD]
};
template <int R, int HD>
inline int64_t kv8_scratch_bytes(int ctas) {
  return (int64_t)ctas * (sizeof(Kv8Part) + 2 * R * (sizeof(float2) + HD * sizeof(float)));
}
template <int R, int HD>
inline Kv8Scratch kv8_scratch(void* ws, int ctas) {
  Kv8Scratch s;
  s.head = reinterpret_cast<Kv8Part*>(ws);
  s.ml = reinterpret_cast<float2*>(s.head + ctas);
  s.o = reinterpret_cast<float*>(s.ml + (int64_t)2 * ctas * R);
  return s;
}

// Softmax factors with a sink: o / l becomes o * result.
MSGL_DEVICE float kv8_norm(float m, float l, const float* sinks, int head) {
  float f = 1.f;
  if (sinks != nullptr && l != 0.f) {
    const float sink = sinks[head] * kKv8Log2e, mn = fmaxf(m, sink);
    f = exp2f(m - mn);
    l = l * f + exp2f(sink - mn);
  }
  return l == 0.f ? 0.f : f / l;
}

// Rows behind the last request's.
template <int HD>
MSGL_DEVICE void kv8_zero_tail(const Kv8Attn& p, int tid, int threads) {
  if (!p.zero_tail) return;
  const int from = min(max(p.cu_q[p.num_reqs], 0), p.total_q);
  const int64_t per = (int64_t)p.nq * HD / 8, end = p.total_q * per;
#pragma unroll 1
  for (int64_t i = from * per + (int64_t)blockIdx.x * threads + tid; i < end; i += (int64_t)gridDim.x * threads)
    reinterpret_cast<uint4*>(p.o)[i] = make_uint4(0, 0, 0, 0);
}

template <int R, int HD>
MSGL_DEVICE void kv8_join_row(const Kv8Attn& p, const Kv8Scratch& s, const Kv8Part& hd, int c, int i, int lane, int G) {
  const int r = hd.r0 + i, tok = kv8_token(p, r), head = hd.h * G + r - tok * G;
  // part 0 ends its CTA's run, the others begin theirs: slots 2 c + 1, 2 (c + 1), 2 (c + 2), ..
  constexpr int E = HD / 32;
  float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int j0 = 0; j0 < hd.parts; j0 += 32) {
    const int n = min(32, hd.parts - j0), j = j0 + lane;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < n) ml = s.ml[(int64_t)(j == 0 ? 2 * c + 1 : 2 * (c + j)) * R + i];
    const float mx = fmaxf(m, warp_max(ml.x)), base = mx == -INFINITY ? 0.f : mx, f = exp2f(m - base), w = exp2f(ml.x - base);
    m = mx;
    l = l * f + w * ml.y;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= f;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const float* src = s.o + ((int64_t)(j0 + k == 0 ? 2 * c + 1 : 2 * (c + j0 + k)) * R + i) * HD + lane * E;
      if constexpr (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src);
        acc[0] += wk * x.x, acc[1] += wk * x.y, acc[2] += wk * x.z, acc[3] += wk * x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(src);
        acc[0] += wk * x.x, acc[1] += wk * x.y;
      }
    }
  }
  const float f = kv8_norm(m, warp_sum(l), p.sinks, head);
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.o) + ((int64_t)(hd.q0 + tok) * p.nq + head) * (HD / 2) + lane * (E / 2);
#pragma unroll
  for (int e = 0; e < E; e += 2) dst[e / 2] = pack_bf16(acc[e] * f, acc[e + 1] * f);
}

// Joins cut segments: grid (ctas, groups of four rows), a warp per row. Few registers and threads, so that its CTAs fit beside the
// last ones of the kernel before it and only its loads are waited for.
template <int R, int HD>
__global__ void __launch_bounds__(128) kv8_join_kernel(Kv8Attn p, Kv8Scratch s) {
  pdl_wait();
  pdl_launch();
  const int c = blockIdx.x, lane = threadIdx.x & 31, G = p.nq / p.nkv;
  const Kv8Part hd = s.head[c];
  if (hd.parts == 0) return;
  for (int i = blockIdx.y * 4 + (threadIdx.x >> 5); i < hd.nr; i += gridDim.y * 4) kv8_join_row<R, HD>(p, s, hd, c, i, lane, G);
}

}  // namespace msgl
