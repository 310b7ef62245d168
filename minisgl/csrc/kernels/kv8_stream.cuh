// Attention over the 8-bit cache for few rows per request and kv head: decoded tokens, a few drafted ones.
//
// What bounds it is the cache's bytes, so the kernel is a stream of them: two CTAs per SM, each two warps that issue
// copies of whole pages (codes swizzled by the tensor map, scales as they lie) into a ring of 64-key stages, and four
// warps that take 16 keys each of every stage. (Two CTAs: while one starts or ends a segment the other streams.) Codes go from
// shared memory to registers once, 16 bytes a lane, in an order of head dims and keys that fits mma.sync without a
// transposition:
//   S^T = K Q^T (m16n8k16, 16 keys x 8 rows): lane (g, t) = (lane / 4, lane % 4) holds of keys g and g + 8 the head dims
//     [HD/4 t, HD/4 (t + 1)): four codes are two registers of one step. The queries' fragments are loaded in the same order.
//   O^T += V^T P^T (16 head dims x 8 rows): lane (g, t) holds of keys 2t, 2t + 1, 2t + 8, 2t + 9 the HD / 8 head dims from
//     HD/8 g on, and pairs of keys are made by byte permutes; P^T's fragments are S^T's, turned by movmatrix in fp16. Lane
//     (g, t) ends up with HD / 8 head dims in a row of rows 2t and 2t + 1.
// Keys as the 16 rows of a product, since the query rows are often 8 at most: NR = 1 takes tiles of 8 rows, NR = 2 of 16.
// Codes are exact in fp16, and the queries are, scaled by a power of two. Logits, sums and O are fp32.
// A warp keeps its own maximum and sum; the four are joined when a segment ends (see kv8_plan.cuh).
//
// Measured (8 kv heads of 128, back to back in a graph): 4 requests of 100000 keys, int8, 148 us or 5.7 TB/s; 128 of 100 to 2048, e4m3,
// 61 us or 4.8 TB/s, of which some 8 us are the plan, the first copies and the join of cut segments (a ring of 3 stages instead
// of 4 takes 62). Two tiles of 16 rows (25 rows of 5 drafted tokens, 16 requests of 6000) take 94 us: there it is two warps a
// scheduler, each waiting for its own products and conversions, that bound it (52% of the issue slots used).
#pragma once
#include "kv8.cuh"
#include "kv8_plan.cuh"

namespace msgl {

constexpr int kKsWarps = 4;   // of products
constexpr int kKsCopies = 2;  // warps that issue copies
constexpr int kKsCost = 3;    // of a segment, in blocks
constexpr int kKsThreads = 32 * (kKsWarps + kKsCopies);
constexpr int kKsDescs = 4;   // segments looked up ahead

struct KsDesc {
  int q0, h, r0, nr, row, pos0, pos1, L, n, lo, kend, blk, nb, slot, parts, valid;  // blocks [blk, blk + nb); slot -1: whole
};

template <int HD, int NR>
struct KsCfg {
  static constexpr int kRows = 8 * NR;
  static constexpr int kTile = kKv8Block * HD;
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = HD == 128 ? 4 : 8;
  static constexpr int kScales = 2 * kKv8Block * 4;  // of a stage: keys', then values'
  // merge scratch: floats of a lane's head dims and of a row (padded, against bank conflicts)
  static constexpr int kMergeQ = HD / 8 + 4, kMergeRow = 8 * kMergeQ + 4;
  static constexpr int kMerge = kKsWarps * kRows * kMergeRow * 4 + kKsWarps * kRows * 8;
  static constexpr int kSmem = 1024 + kStages * (kStage + kScales) + kMerge + kKsDescs * (int)sizeof(KsDesc) + (int)sizeof(Kv8Plan) +
                               8 * (kKsThreads / 32) + 8 * (2 * kStages + 2 * kKsDescs) + 16;
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs per SM");
};

// byte of (row, 16-byte chunk) in a tile of HD-byte rows as the tensor map's swizzle lays it out
template <int HD>
MSGL_DEVICE uint32_t ks_swz(int row, int chunk) {
  return HD == 128 ? (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)) : (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
}
MSGL_DEVICE void ks_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HD, bool FP8, int NR>
__global__ void __launch_bounds__(kKsThreads, 2)
kv8_stream_kernel(const __grid_constant__ CUtensorMap tc, const __grid_constant__ CUtensorMap ts, Kv8Attn p, Kv8Order order, Kv8Scratch scratch) {
  using C = KsCfg<HD, NR>;
  constexpr int NK = HD / 16;  // steps of K Q^T, and tiles of O^T
  constexpr int R = C::kRows;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* scales = reinterpret_cast<float*>(ring + C::kStages * C::kStage);
  float* merge = scales + C::kStages * (C::kScales / 4);                       // [warps][16][kMergeRow]
  float2* merge_ml = reinterpret_cast<float2*>(merge + kKsWarps * R * C::kMergeRow);  // [warps][16]
  KsDesc* descs = reinterpret_cast<KsDesc*>(merge_ml + kKsWarps * R);
  Kv8Plan* plan = reinterpret_cast<Kv8Plan*>(descs + kKsDescs);
  int64_t* red = reinterpret_cast<int64_t*>(plan + 1);
  uint64_t* full = reinterpret_cast<uint64_t*>(red + kKsThreads / 32);
  uint64_t* empty = full + C::kStages;
  uint64_t* dfull = empty + C::kStages;
  uint64_t* dempty = dfull + kKsDescs;
  volatile int* abort_flag = reinterpret_cast<int*>(dempty + kKsDescs);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kKsWarps);
    }
#pragma unroll 1
    for (int i = 0; i < kKsDescs; ++i) {
      mbar_init(&dfull[i], 1);
      mbar_init(&dempty[i], kKsWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tc);
    prefetch_tmap(&ts);
  }
  pdl_wait();
  pdl_launch();
  if (threadIdx.x == 0) scratch.head[blockIdx.x].parts = 0;
  kv8_plan<kKsCost, kKsThreads>(p, R, kKsCost + 2, plan, red);  // (its barriers order the initialisation above as well)
  const Kv8Plan pl = *plan;
  const int G = p.nq / p.nkv;
  kv8_zero_tail<HD>(p, threadIdx.x, kKsThreads);

  if (warp >= kKsWarps) {
    // ------------------------------------------------------------------ segments and copies
    // Every copying warp goes through the run's segments and takes every second block; the first one publishes them.
    const int me = warp - kKsWarps;
    const int page = p.page, gpb = kKv8Block / page, mine = 32 / gpb;  // pages of a block, blocks whose slots the lanes hold
    int b = pl.b, h = pl.h, t = pl.t, tiles = 0;
    uint32_t seq = 0;
    int64_t u = pl.u0, s0 = pl.s0;
    bool ok = true;
    Kv8Req r = pl.r;
    if (u < pl.u1) tiles = kv8_tiles(r, G, R);
    int i = 0, issued = 0;
    uint32_t last = 0;
#pragma unroll 1
    for (; ok && u < pl.u1; ++i) {
      const Kv8Tile k = kv8_tile(p, r, G, R, t);
      // blocks [from, to) of the segment: its first kKsCost units are none
      const int from = (int)max(u - s0 - kKsCost, (int64_t)0), to = (int)min((int64_t)k.nblk, pl.u1 - s0 - kKsCost);
      if (to <= 0) break;  // (the run ends before the segment's first block)
      if (me == 0) {
        const int d = i % kKsDescs;
        if (lane == 0) {
          ok = kv8_wait(&dempty[d], ((i / kKsDescs) & 1) ^ 1);
          if (ok) {
            const bool starts = from == 0, ends = to == k.nblk;
            KsDesc& D = descs[d];
            D.q0 = r.q0; D.h = h; D.r0 = k.r0; D.nr = k.nr; D.row = r.row; D.pos0 = k.pos0; D.pos1 = k.pos1; D.L = r.L; D.n = r.n;
            D.lo = k.lo; D.kend = k.kend; D.blk = k.blk0 + from; D.nb = to - from; D.valid = 1;
            D.slot = starts && ends ? -1 : starts ? 2 * (int)blockIdx.x + 1 : 2 * (int)blockIdx.x;
            const int parts = starts && !ends ? kv8_cta_of(pl, s0 + kKsCost + k.nblk - 1) - (int)blockIdx.x + 1 : 0;
            if (parts > 0) {  // (the run's last segment)
              Kv8Part& hd = scratch.head[blockIdx.x];
              hd.q0 = r.q0; hd.r0 = k.r0; hd.nr = k.nr; hd.h = h; hd.parts = parts;
            }
            mbar_arrive(&dfull[d]);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
      } else if (lane < k.nr) {  // the segment's queries are wanted when the ones before it are done
        const int rr = k.r0 + lane, tok = kv8_token(p, rr);
        const char* src = reinterpret_cast<const char*>(p.q) + 2 * ((r.q0 + tok) * p.q_row + (int64_t)(h * G + rr - tok * G) * p.q_head);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
        if (HD == 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + 128));
      }
      // This warp's blocks j = j0, j0 + 2, ..: their pages' slots, a batch of `mine` blocks ahead. Looked up in one go, looked over
      // when their turn comes, so that the loads' latency is not waited for.
      const int page0 = (k.blk0 + from) * gpb, pages_end = k.kend > k.lo ? (k.kend - 1) / page + 1 : 0;
      const int j0 = (int)((me - seq) & (kKsCopies - 1));
      auto look_up = [&](int j) {
        const int g = page0 + (j + lane / gpb * kKsCopies) * gpb + lane % gpb;
        return g < pages_end && j + lane / gpb * kKsCopies < to - from ? p.page_table[(int64_t)r.row * p.pt_stride + (int64_t)g * page] : -1;
      };
      int next = look_up(j0), slots = -1;
#pragma unroll 1
      for (int j = j0, at = 0; j < to - from; j += kKsCopies, ++at) {
        if (at % mine == 0) {
          slots = next;
          const int g = page0 + (j + lane / gpb * kKsCopies) * gpb + lane % gpb;
          if (g < pages_end && j + lane / gpb * kKsCopies < to - from) slots = kv8_checked(p, slots);
          if (j + mine * kKsCopies < to - from) next = look_up(j + mine * kKsCopies);
        }
        const uint32_t x = seq + j, stage = x % C::kStages;
        ok = kv8_wait_warp(&empty[stage], ((x / C::kStages) & 1) ^ 1);
        if (!ok) break;
        const int pages = max(0, min(gpb, pages_end - (page0 + j * gpb)));
        kv8_copy_block<HD, 4>(p, &tc, &ts, ring + stage * C::kStage, scales + stage * (C::kScales / 4), &full[stage], h, slots,
                           at % mine * gpb, pages);
        last = x;
        ++issued;
      }
      if (!ok) break;
      seq += to - from;
      // the next segment
      u = s0 + kKsCost + to;
      s0 += kKsCost + k.nblk;
      if (u < pl.u1 && ++t == tiles) {
        t = 0;
        if (++h == p.nkv) {
          h = 0;
          do {
            if (++b >= p.num_reqs) break;  // (never: units are left)
            r = kv8_request(p, b);
            tiles = kv8_tiles(r, G, R);
          } while (tiles == 0);
          if (b >= p.num_reqs) u = pl.u1;
        }
      }
    }
    if (ok) {
      if (me == 0 && lane == 0 && kv8_wait(&dempty[i % kKsDescs], ((i / kKsDescs) & 1) ^ 1)) {
        descs[i % kKsDescs].valid = 0;
        mbar_arrive(&dfull[i % kKsDescs]);
      }
    } else if (lane == 0) {  // given up: this warp's copies in flight land before the CTA's memory goes
      kv8_gave_up(700);
#pragma unroll 1
      for (int n = 0; n < min(issued, C::kStages / kKsCopies); ++n) {
        const uint32_t x = last - n * kKsCopies;
        kv8_wait(&full[x % C::kStages], (x / C::kStages) & 1);
      }
    }
    return;
  }

  // -------------------------------------------------------------------- products
  const int g = lane >> 2, t = lane & 3, key0 = warp * 16;
  const int ctid = threadIdx.x;
  // this warp's keys lie in one page: [keys' page][values' page] each
  const int base = key0 + (key0 & ~(p.page - 1));
  const uint32_t k_at = (uint32_t)(base + order.codes * p.page) * HD, v_at = (uint32_t)(base + (order.codes ^ 1) * p.page) * HD;
  const uint32_t ks_at = (uint32_t)(base + order.scales * p.page + g) * 4, vs_at = (uint32_t)(base + (order.scales ^ 1) * p.page + g) * 4;
  uint32_t seq = 0;  // stages gone through
  bool dead = false;
#pragma unroll 1
  for (int i = 0;; ++i) {
    const int d = i % kKsDescs;
    if (!dead && !kv8_wait_warp(&dfull[d], (i / kKsDescs) & 1)) { dead = true; *abort_flag = 1; }
    if (!dead && !descs[d].valid) {
      named_bar_sync(1, kKsWarps * 32);  // (pairs with the barrier below of a warp that has given up)
      break;
    }
    const KsDesc D = descs[d];
    __syncwarp();
    if (!dead && lane == 0) mbar_arrive(&dempty[d]);

    // queries: rows g (+ 8) in fragments, brought to fp16's range by a power of two each
    uint32_t qf[NR][NK][2];
    float qs[NR][2];  // of rows 2 t and 2 t + 1
    int qpos[NR][2];
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      const int rr = g + 8 * x, r = D.r0 + rr, tok = kv8_token(p, r);
      const bool in = !dead && rr < D.nr;
      uint4 u[HD / 32];
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) u[j] = make_uint4(0, 0, 0, 0);
      if (in) {
        const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(p.q) + (D.q0 + tok) * p.q_row +
                                   (int64_t)(D.h * G + r - tok * G) * p.q_head + t * (HD / 4);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) u[j] = __ldg(reinterpret_cast<const uint4*>(src) + j);
      }
      const int pos = in ? D.L - D.n + tok : -1;
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < HD / 32; ++j)
        m = __vmaxu2(m, __vmaxu2(__vmaxu2(u[j].x & 0x7fff7fffu, u[j].y & 0x7fff7fffu), __vmaxu2(u[j].z & 0x7fff7fffu, u[j].w & 0x7fff7fffu)));
      m = max(m & 0xffffu, m >> 16);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const float f = kv8_q_factor(__uint_as_float(m << 16));
      const float back = p.scale * kKv8Log2e * kv8_reciprocal(f);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qs[x][e] = __shfl_sync(0xffffffffu, back, (2 * t + e) * 4);
        qpos[x][e] = __shfl_sync(0xffffffffu, pos, (2 * t + e) * 4);
      }
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) {
        const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)  // dims 8 j + 2 e and the next: step 2 j + e / 2
          qf[x][2 * j + (e >> 1)][e & 1] = pack_half(bf16_lo(w[e]) * f, bf16_hi(w[e]) * f);
      }
    }

    float m[NR][2], l[NR][2], o[NR][NK][4];
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      m[x][0] = m[x][1] = -INFINITY;
      l[x][0] = l[x][1] = 0.f;
#pragma unroll
      for (int j = 0; j < NK; ++j) o[x][j][0] = o[x][j][1] = o[x][j][2] = o[x][j][3] = 0.f;
    }

#pragma unroll 1
    for (int j = 0; j < D.nb && !dead; ++j) {
      const uint32_t at = seq + j, stage = at % C::kStages;
      if (!kv8_wait_warp(&full[stage], (at / C::kStages) & 1)) { dead = true; *abort_flag = 1; break; }
      const uint8_t* st = ring + stage * C::kStage;
      const uint8_t* sc = reinterpret_cast<const uint8_t*>(scales) + stage * C::kScales;
      // S^T of keys g and g + 8 (c = 0, 1), rows 2 t and 2 t + 1 (e): s[x][2 c + e]
      float s[NR][4], ksc[2], vsc[2];
      {
        uint32_t w[2][NK];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int y = 0; y < HD / 64; ++y) {
            const uint4 v = *reinterpret_cast<const uint4*>(st + k_at + ks_swz<HD>(8 * c + g, t * (HD / 64) + y));
            w[c][4 * y] = v.x; w[c][4 * y + 1] = v.y; w[c][4 * y + 2] = v.z; w[c][4 * y + 3] = v.w;
          }
          ksc[c] = *reinterpret_cast<const float*>(sc + ks_at + 32 * c);
          vsc[c] = *reinterpret_cast<const float*>(sc + vs_at + 32 * c);
        }
        float s2[NR][4];  // (two sums each)
#pragma unroll
        for (int x = 0; x < NR; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][e] = s2[x][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          uint32_t a[4];
          kv8_to_half<FP8>(w[0][kk], a[0], a[2]);
          kv8_to_half<FP8>(w[1][kk], a[1], a[3]);
#pragma unroll
          for (int x = 0; x < NR; ++x) ks_mma(kk & 1 ? s2[x] : s[x], a, qf[x][kk][0], qf[x][kk][1]);
        }
#pragma unroll
        for (int x = 0; x < NR; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][e] = (s[x][e] + s2[x][e]) * ksc[e >> 1] * qs[x][e & 1];
      }
      const int k0 = (D.blk + j) * kKv8Block + key0, k1 = k0 + 16;
      const bool inside = k1 <= D.pos0 + 1 && (p.window <= 0 || k0 >= D.pos1 - p.window + 1);  // every row sees every key
      if (!inside) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int kp = k0 + 8 * c + g;
#pragma unroll
          for (int x = 0; x < NR; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const bool seen = kp <= qpos[x][e] && (p.window <= 0 || kp > qpos[x][e] - p.window);
              s[x][2 * c + e] = seen ? s[x][2 * c + e] : -INFINITY;
            }
          if (kp < D.lo || kp >= D.kend) vsc[c] = 0.f;  // (it may be no position at all: its scale can be anything)
        }
      }
      const float lv[2] = {kv8_log_scale(vsc[0]), kv8_log_scale(vsc[1])};
      // running offsets and sums
      float f[NR][2];
      uint32_t pf[NR][2];
      bool grown = false;
#pragma unroll
      for (int x = 0; x < NR; ++x) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(s[x][e] + lv[0], s[x][2 + e] + lv[1]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          mx = fmaxf(mx - kKv8Top, m[x][e]);
          const float base = mx == -INFINITY ? 0.f : mx;
          f[x][e] = kv8_exp2(m[x][e] - base);
          grown |= mx != m[x][e];
          m[x][e] = mx;
          float sum = 0.f;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float y = s[x][2 * c + e], w = kv8_exp2(y - base);
            sum += w;
            s[x][2 * c + e] = y == -INFINITY ? 0.f : w * vsc[c];  // (a hidden key's weight is zero whatever its scale)
          }
          l[x][e] = l[x][e] * f[x][e] + sum;  // (of this lane's keys; joined over g at the end)
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
          asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pf[x][c]) : "r"(pack_half(s[x][2 * c], s[x][2 * c + 1])));
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int x = 0; x < NR; ++x)
#pragma unroll
          for (int n = 0; n < NK; ++n) {
            o[x][n][0] *= f[x][0]; o[x][n][1] *= f[x][1]; o[x][n][2] *= f[x][0]; o[x][n][3] *= f[x][1];
          }
      }
      // O^T: tile n holds head dims HD/8 g + 2 n and the next
      {
        uint32_t vw[4][NK / 2];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = 2 * t + (e & 1) + 8 * (e >> 1);
          if constexpr (HD == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(st + v_at + ks_swz<HD>(key, g));
            vw[e][0] = v.x; vw[e][1] = v.y; vw[e][2] = v.z; vw[e][3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(st + v_at + ks_swz<HD>(key, g >> 1) + (g & 1) * 8);
            vw[e][0] = v.x; vw[e][1] = v.y;
          }
          const int kp = k0 + key;
          if (!inside && (kp < D.lo || kp >= D.kend)) {  // (nor are such a key's codes any)
#pragma unroll
            for (int c = 0; c < NK / 2; ++c) vw[e][c] = 0u;
          }
        }
#pragma unroll
        for (int c = 0; c < NK / 2; ++c) {
          uint32_t b[2][4];  // head dims 4 c .. 4 c + 3 of keys 2 t, 2 t + 1 and of the other two
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t lo = __byte_perm(vw[2 * x][c], vw[2 * x + 1][c], 0x5140), hi = __byte_perm(vw[2 * x][c], vw[2 * x + 1][c], 0x7362);
            kv8_to_half<FP8>(lo, b[x][0], b[x][1]);
            kv8_to_half<FP8>(hi, b[x][2], b[x][3]);
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint32_t a[4] = {b[0][2 * n], b[0][2 * n + 1], b[1][2 * n], b[1][2 * n + 1]};
#pragma unroll
            for (int x = 0; x < NR; ++x) ks_mma(o[x][2 * c + n], a, pf[x][0], pf[x][1]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
    }
    seq += D.nb;

    // join the warps
#pragma unroll
    for (int x = 0; x < NR; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], 4);
        l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], 8);
        l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], 16);
        const int rr = 8 * x + 2 * t + e;
        if (rr < D.nr) {
          if (g == 0) merge_ml[warp * R + rr] = make_float2(m[x][e], l[x][e]);
          float* dst = merge + (warp * R + rr) * C::kMergeRow + g * C::kMergeQ;
#pragma unroll
          for (int n = 0; n < NK; n += 2)
            *reinterpret_cast<float4*>(dst + 2 * n) = make_float4(o[x][n][e], o[x][n][2 + e], o[x][n + 1][e], o[x][n + 1][2 + e]);
        }
      }
    named_bar_sync(1, kKsWarps * 32);
    if (*abort_flag) {
      if (dead) kv8_gave_up(710);
      break;
    }
#pragma unroll 1
    for (int idx = ctid; idx < D.nr * (HD / 4); idx += kKsWarps * 32) {
      const int rr = idx / (HD / 4), c4 = idx % (HD / 4);
      float mx = -INFINITY;
      float2 ml[kKsWarps];
#pragma unroll
      for (int w = 0; w < kKsWarps; ++w) {
        ml[w] = merge_ml[w * R + rr];
        mx = fmaxf(mx, ml[w].x);
      }
      const float base = mx == -INFINITY ? 0.f : mx;
      float ll = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kKsWarps; ++w) {
        const float fw = kv8_exp2(ml[w].x - base);
        ll += fw * ml[w].y;
        const float4 v = *reinterpret_cast<const float4*>(merge + (w * R + rr) * C::kMergeRow + c4 / (HD / 32) * C::kMergeQ + c4 % (HD / 32) * 4);
        acc.x += fw * v.x; acc.y += fw * v.y; acc.z += fw * v.z; acc.w += fw * v.w;
      }
      if (D.slot < 0) {
        const int r = D.r0 + rr, tok = kv8_token(p, r), head = D.h * G + r - tok * G;
        const float f = kv8_norm(mx, ll, p.sinks, head);
        reinterpret_cast<uint2*>(p.o)[((int64_t)(D.q0 + tok) * p.nq + head) * (HD / 4) + c4] =
            make_uint2(pack_bf16(acc.x * f, acc.y * f), pack_bf16(acc.z * f, acc.w * f));
      } else {
        const int64_t row = (int64_t)D.slot * R + rr;
        reinterpret_cast<float4*>(scratch.o)[row * (HD / 4) + c4] = acc;
        if (c4 == 0) scratch.ml[row] = make_float2(mx, ll);
      }
    }
    named_bar_sync(1, kKsWarps * 32);  // the merge scratch is free
  }
}

}  // namespace msgl
