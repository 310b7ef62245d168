// Attention over the 8-bit cache for many rows per request and kv head: chunks of prompts, drafted tokens of wide groups.
//
// One CTA per SM takes segments of up to 256 packed rows (see kv8_plan.cuh), two tiles of up to 128 rows, whole tokens each,
// that share every key and value block, 64 keys at a time, on the 5th-generation tensor core:
//
//   warp 0        goes through the run's segments, publishes them, copies raw pages into a ring by TMA
//   warps 1, 2    issue the products of one tile each: S = Q K^T a block ahead, and, once the weights are there, O += P V, P out
//                 of tensor memory
//   warp 3        copies the segments' queries, as they are, by TMA
//   warps 4 - 11  softmax, 32 rows a warp, four rows and 16 keys a lane: S out of tensor memory, weights as fp16 over S's columns, O rescaled there
//                 when a row's offset grows by more than 2^(15 - kKtTop), O read out and written at the segment's end
//   warps 12 - 15 convert codes to operand tiles, once for both tiles of rows: keys to bf16, which is the queries' type, values to
//                 fp16, which has the more bits for the weights (exact, both), and scales to what the softmax wants of them
//
// A block's S and its weights share 64 columns of tensor memory, and each tile has two such: S 2 x 2 x 64 columns, O 2 x 128. (With
// Q in tensor memory instead of shared memory there is room for one only; less shared memory is read then, but a tile's
// softmax waits for its products some 1200 cycles every block, which the other tile does not fill.)
//
// Numerics as in kv8_stream.cuh, with kKtTop for kKv8Top: room for offsets that are not moved at every block.
//
// Measured (40 heads over 8 of 128): a chunk of 2048 tokens after 30000 cached ones takes 1520 us in int8, 856 TFLOP/s, before the
// power limit lowers the clock; 28 prompts of 100 to 1024 tokens 302 us in e4m3. A block of 256 x 64 takes some 2700 cycles, of which the tensor core is busy for 40%; the
// softmax has 2100 of work (half of it waits for the 2^x units and issue slots that two of its warps share with a converting one), and
// the rest is its wait for S. Code that few blocks run costs its way from the L2 cache each time, hence the loops in it.
#pragma once
#include "kv8.cuh"
#include "kv8_plan.cuh"

#include <limits.h>

namespace msgl {

constexpr int kKtRows = 256;
constexpr int kKtThreads = 512;
constexpr int kKtCost = 3;      // of a segment, in blocks
constexpr int kKtDescs = 4;     // segments looked up ahead
constexpr int kKtSlots = 8;     // of scales
// Offsets are moved where a weight would pass 2^15, so 2^9 lie between the largest one seen when they were set and that. (2^5 of
// room has a warp's 32 rows move in half of the first blocks of short prompts: 368 us instead of 320 for 28 prompts of 100 to
// 1024 tokens. fp16 then rounds weights to 2^-31 of the largest one at worst.)
constexpr float kKtTop = 6.f;
constexpr int kKtConv = 12, kKtSoft = 4;  // first warps of the converters and of the softmax
// registers of a thread in warps 0 - 3, the softmax and the converters: of the launch's 4 x 128 a row of warps
constexpr int kKtRegs = 128, kKtRegsFew = 64, kKtRegsSoft = 176, kKtRegsConv = 96;
static_assert(kKtRegsFew + 2 * kKtRegsSoft + kKtRegsConv <= 4 * kKtRegs, "more registers than the launch has");
template <int N>
MSGL_DEVICE void kt_fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
MSGL_DEVICE void kt_more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

struct KtDesc {
  int q0, h, r0, nr, L, n, lo, kend, blk, nb, slot;  // nb 0: no more
  int pad;
};
struct KtScales {
  float ks[kKv8Block], lv[kKv8Block], vs[kKv8Block];
  uint32_t bad[4];  // bit c % 32 of word c / 32: key c has no finite scale (0 stands in its place)
};

template <int HD>
struct KtCfg {
  static constexpr int kHalf = kKv8Block * 128;      // a block's 64 head dims as an fp16 operand
  static constexpr int kTile = kHalf * (HD / 64);
  static constexpr int kStages = 3;                  // of K and of V operands
  static constexpr int kRaw = HD == 128 ? 3 : 8;     // of codes
  static constexpr int kRawStage = 2 * kKv8Block * HD;
  static constexpr int kRawScales = 2 * kKv8Block * 4;
  static constexpr int kQHalf = 128 * 128, kQTile = kQHalf * (HD / 64);  // a tile's queries
  static constexpr int kOffQ = 2 * kStages * kTile;
  static constexpr int kOffRaw = kOffQ + 2 * kQTile;
  static constexpr int kOffSc = kOffRaw + kRaw * kRawStage;
  static constexpr int kOffSlots = kOffSc + kRaw * kRawScales;
  static constexpr int kOffDesc = kOffSlots + kKtSlots * (int)sizeof(KtScales);
  static constexpr int kOffPlan = kOffDesc + kKtDescs * (int)sizeof(KtDesc);
  static constexpr int kOffRed = kOffPlan + (int)sizeof(Kv8Plan);
  static constexpr int kOffBars = kOffRed + 8 * (kKtThreads / 32);
  static constexpr int kBars = 4 * kStages + 2 * kRaw + kKtSlots + 2 * kKtDescs + 2 + 3 * 4 + 2;
  static constexpr int kSmem = 1024 + kOffBars + 8 * kBars + 16;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  // tensor memory columns
  static constexpr int kS = 0, kO = 256;
};

constexpr uint32_t kt_idesc(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }  // fp16 operands, fp32 sums

MSGL_DEVICE void kt_prefetch_3d(const CUtensorMap* map, int x, int y, int z) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// 16 lanes x 64 columns of tensor memory as mma's accumulators lie: lane (g, t) = (lane / 4, lane % 4) holds of rows g
// (registers 4n, 4n + 1) and g + 8 (4n + 2, 4n + 3) the columns 8n + 2t and the next.
MSGL_DEVICE void kt_load_s(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// 16 lanes x 32 columns in the same order: lane (g, t) holds column 4n + t of rows g (register 2n) and g + 8 (2n + 1): fp16
// pairs of those S.
MSGL_DEVICE void kt_store_p(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// The same for 32 columns, for 16 columns of S and 8 of its weights.
MSGL_DEVICE void kt_load_o(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
}
MSGL_DEVICE void kt_load_s16(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
MSGL_DEVICE void kt_store_p8(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}

// A lane's four rows, 8 apart: their positions, running offsets and this lane's part of their sums, and what their O has to be
// multiplied by first.
struct KtRows {
  int pos[4];
  float m[4], l[4], alpha[4];
};
// The keys of a block, [first, end), that they see (worked out where a block is seen in part: eight registers less for the others).
struct KtSeen {
  int first[4], end[4];
  MSGL_DEVICE KtSeen(const KtRows& w, int k0, int window, bool part) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      first[k] = part && window > 0 ? max(0, w.pos[k] - window + 1 - k0) : 0;
      end[k] = !part ? kKv8Block : w.pos[k] < k0 ? 0 : min(w.pos[k] - k0, kKv8Block - 1) + 1;
    }
  }
};

// Offsets with which the largest weight of this block is 2^kKtTop (see kKv8Top), for the rows that have a lower one. (A compact loop, like all that not every block needs: unrolled it comes out of L2 each time, and takes ten times as long.)
MSGL_DEVICE void kt_move(uint32_t s_tmem, const KtScales& sc, KtRows& w, const KtSeen& seen, float qs, int t) {
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
  for (int n = 0; n < kKv8Block; n += 16) {
    uint32_t u[2][8];
    kt_load_s16(s_tmem + n, u[0]);
    kt_load_s16(s_tmem + n + (16u << 16), u[1]);
    tc_wait_ld();
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int c = n + 8 * y + 2 * t;
      const float2 ks = *reinterpret_cast<const float2*>(&sc.ks[c]), lv = *reinterpret_cast<const float2*>(&sc.lv[c]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t* s = &u[k >> 1][4 * y + 2 * (k & 1)];
        const float a = fmaf(__uint_as_float(s[0]) * ks.x, qs, lv.x), b = fmaf(__uint_as_float(s[1]) * ks.y, qs, lv.y);
        if (c >= seen.first[k] && c < seen.end[k]) top[k] = fmaxf(top[k], a);
        if (c + 1 >= seen.first[k] && c + 1 < seen.end[k]) top[k] = fmaxf(top[k], b);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
    top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 2)) - kKtTop;
    if (top[k] > w.m[k]) {
      const float f = kv8_exp2(w.m[k] - top[k]);
      w.m[k] = top[k];
      w.l[k] *= f;
      w.alpha[k] *= f;
    }
  }
}

// The weights of a block that some of the lane's rows see in part only, over S's columns.
MSGL_DEVICE void kt_weights_in_part(uint32_t s_tmem, const KtScales& sc, KtRows& w, const KtSeen& seen, float qs, int t) {
#pragma unroll 1
  for (int n = 0; n < kKv8Block; n += 16) {
    uint32_t u[2][8], pk[2][4];
    kt_load_s16(s_tmem + n, u[0]);
    kt_load_s16(s_tmem + n + (16u << 16), u[1]);
    tc_wait_ld();
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int c = n + 8 * y + 2 * t;
      const float2 ks = *reinterpret_cast<const float2*>(&sc.ks[c]), vs = *reinterpret_cast<const float2*>(&sc.vs[c]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t* s = &u[k >> 1][4 * y + 2 * (k & 1)];
        const float base = w.m[k] == -INFINITY ? 0.f : w.m[k];
        float a = kv8_exp2(fmaf(__uint_as_float(s[0]) * ks.x, qs, -base)), b = kv8_exp2(fmaf(__uint_as_float(s[1]) * ks.y, qs, -base));
        if (!(c >= seen.first[k] && c < seen.end[k])) a = 0.f;
        if (!(c + 1 >= seen.first[k] && c + 1 < seen.end[k])) b = 0.f;
        w.l[k] += a + b;
        pk[k >> 1][2 * y + (k & 1)] = pack_half(a * vs.x, b * vs.y);
      }
    }
    // (the columns it overwrites have been read: keys n / 2 .. n / 2 + 7)
    kt_store_p8(s_tmem + n / 2, pk[0]);
    kt_store_p8(s_tmem + n / 2 + (16u << 16), pk[1]);
  }
}

// The weights of a block that every row sees, as fp16 pairs, with the offsets as they are, and this lane's sums of 2^(s_j - m).
// Returns whether a weight is beyond 2^15, or a sum beyond 2^108 (keys whose values are nearly nothing).
MSGL_DEVICE bool kt_weights(uint32_t s_tmem, const KtScales& sc, const KtRows& w, float qs, int t, float (&sum)[4], uint32_t (&pk)[2][16]) {
  uint32_t u[2][32];
  kt_load_s(s_tmem, u[0]);
  kt_load_s(s_tmem + (16u << 16), u[1]);
  const uint64_t q2 = f2_pack(qs, qs);
  uint64_t b2[4], total[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float base = w.m[k] == -INFINITY ? 0.f : w.m[k];
    b2[k] = f2_pack(-base, -base);
    total[k] = 0;
  }
  __half2 top = __float2half2_rn(0.f);
  tc_wait_ld();
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const int c = 8 * n + 2 * t;
    const uint64_t ks = *reinterpret_cast<const uint64_t*>(&sc.ks[c]), vs = *reinterpret_cast<const uint64_t*>(&sc.vs[c]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t* s = &u[k >> 1][4 * n + 2 * (k & 1)];
      const float2 x = f2_unpack(f2_fma(f2_mul(f2_pack(__uint_as_float(s[0]), __uint_as_float(s[1])), ks), q2, b2[k]));
      const uint64_t e2 = f2_pack(kv8_exp2(x.x), kv8_exp2(x.y));
      total[k] = f2_add(total[k], e2);
      const float2 v = f2_unpack(f2_mul(e2, vs));
      const uint32_t h = pack_half(v.x, v.y);
      top = __hmax2(top, *reinterpret_cast<const __half2*>(&h));
      pk[k >> 1][2 * n + (k & 1)] = h;
    }
  }
  bool beyond = !__hble2(top, __float2half2_rn(32768.f));
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 a = f2_unpack(total[k]);
    sum[k] = a.x + a.y;
    beyond |= !(sum[k] <= 0x1p+108f);
  }
  return beyond;
}

// A block of the lane's rows, which see all of it or (`part`) not: their weights over S's columns. New offsets first where rows
// have none (`fresh`: they have seen no key yet), or weights beyond fp16: few blocks need any, and the others are spared the
// maximum of their logits. Returns whether the rows have got factors for O.
MSGL_DEVICE bool kt_softmax(uint32_t s_tmem, const KtScales& sc, KtRows& w, float qs, int t, int k0, int window, bool part, bool fresh) {
  float sum[4];
  uint32_t pk[2][16];
  bool move = part || fresh, moved = false;
#pragma unroll 1
  for (;;) {
    if (move) {
      const KtSeen seen(w, k0, window, part);
#pragma unroll
      for (int k = 0; k < 4; ++k) w.alpha[k] = 1.f;
      kt_move(s_tmem, sc, w, seen, qs, t);
      moved = true;
      if (part) {
        kt_weights_in_part(s_tmem, sc, w, seen, qs, t);
        return true;
      }
    }
    const bool beyond = kt_weights(s_tmem, sc, w, qs, t, sum, pk);
    if (moved || !__any_sync(0xffffffffu, beyond)) break;
    move = true;
  }
  kt_store_p(s_tmem, pk[0]);
  kt_store_p(s_tmem + (16u << 16), pk[1]);
#pragma unroll
  for (int k = 0; k < 4; ++k) w.l[k] += sum[k];
  return moved;
}

template <int HD, bool FP8>
__global__ void __launch_bounds__(kKtThreads, 1)
kv8_tiles_kernel(const __grid_constant__ CUtensorMap tc, const __grid_constant__ CUtensorMap ts, const __grid_constant__ CUtensorMap tq, Kv8Attn p, Kv8Order order, Kv8Scratch scratch) {
  using C = KtCfg<HD>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sK = smem;
  uint8_t* sV = smem + C::kStages * C::kTile;
  uint8_t* raw = smem + C::kOffRaw;
  float* raw_scales = reinterpret_cast<float*>(smem + C::kOffSc);
  KtScales* slots = reinterpret_cast<KtScales*>(smem + C::kOffSlots);
  KtDesc* descs = reinterpret_cast<KtDesc*>(smem + C::kOffDesc);
  Kv8Plan* plan = reinterpret_cast<Kv8Plan*>(smem + C::kOffPlan);
  int64_t* red = reinterpret_cast<int64_t*>(smem + C::kOffRed);
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
  uint64_t* kempty = kfull + C::kStages;
  uint64_t* vfull = kempty + C::kStages;
  uint64_t* vempty = vfull + C::kStages;
  uint64_t* rfull = vempty + C::kStages;
  uint64_t* rempty = rfull + C::kRaw;
  uint64_t* scfull = rempty + C::kRaw;
  uint64_t* dfull = scfull + kKtSlots;
  uint64_t* dempty = dfull + kKtDescs;
  uint64_t* qfull = dempty + kKtDescs;
  uint64_t* qempty = qfull + 1;
  uint64_t* sfull = qempty + 1;  // [tile][buffer]: S is there
  uint64_t* pfull = sfull + 4;   // its weights are
  uint64_t* pvdone = pfull + 4;  // O holds them, S's columns are free
  uint64_t* ofree = pvdone + 4;  // [tile]: O has been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ofree + 2);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (a warp's number, known as one)
  if (warp == 1) {
    if (lane == 0) {
#pragma unroll 1
      for (int i = 0; i < C::kStages; ++i) {
        mbar_init(&kfull[i], 4);
        mbar_init(&kempty[i], 2);
        mbar_init(&vfull[i], 4);
        mbar_init(&vempty[i], 2);
      }
#pragma unroll 1
      for (int i = 0; i < C::kRaw; ++i) {
        mbar_init(&rfull[i], 1);
        mbar_init(&rempty[i], 4);
      }
#pragma unroll 1
      for (int i = 0; i < kKtSlots; ++i) mbar_init(&scfull[i], 4);
#pragma unroll 1
      for (int i = 0; i < kKtDescs; ++i) {
        mbar_init(&dfull[i], 1);
        mbar_init(&dempty[i], 2 + 1 + 8 + 4);
      }
      mbar_init(qfull, 1);
      mbar_init(qempty, 2);
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        mbar_init(&sfull[i], 1);
        mbar_init(&pfull[i], 4);
        mbar_init(&pvdone[i], 1);
      }
#pragma unroll 1
      for (int i = 0; i < 2; ++i) mbar_init(&ofree[i], 4);
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  } else if (warp == 0 && lane == 0) {
    prefetch_tmap(&tc);
    prefetch_tmap(&ts);
    prefetch_tmap(&tq);
  }
  const int G = p.nq / p.nkv, tokens = 128 / G, trows = tokens * G, R = 2 * trows;  // of a tile, of a segment
#pragma unroll 1
  for (int i = threadIdx.x; i < (128 - trows) * 8 * 2 * (HD / 64); i += kKtThreads) {  // rows that no query is copied to
    const int half = i / ((128 - trows) * 8), at = i % ((128 - trows) * 8);
    *reinterpret_cast<uint4*>(smem + C::kOffQ + half * C::kQHalf + trows * 128 + at * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_wait();
  pdl_launch();
  if (threadIdx.x == 0) scratch.head[blockIdx.x].parts = 0;
  kv8_plan<kKtCost, kKtThreads>(p, R, kKtCost + 2, plan, red);
  const Kv8Plan pl = *plan;
  kv8_zero_tail<HD>(p, threadIdx.x, kKtThreads);

  if (warp == 0) {
    // ------------------------------------------------------------------ segments and copies
    kt_fewer_regs<kKtRegsFew>();
    const int page = p.page, gpb = kKv8Block / page, mine = 32 / gpb;  // pages of a block, blocks whose slots the lanes hold
    int b = pl.b, h = pl.h, t = pl.t, tiles = 0, i = 0;
    uint32_t seq = 0;
    int64_t u = pl.u0, s0 = pl.s0;
    bool ok = true;
    Kv8Req r = pl.r;
    if (u < pl.u1) tiles = kv8_tiles(r, G, R);
#pragma unroll 1
    for (; ok && u < pl.u1; ++i) {
      const Kv8Tile k = kv8_tile(p, r, G, R, t);
      // blocks [from, to) of the segment: its first kKtCost units are none
      const int from = (int)max(u - s0 - kKtCost, (int64_t)0), to = (int)min((int64_t)k.nblk, pl.u1 - s0 - kKtCost);
      if (to <= 0) break;  // (the run ends before the segment's first block)
      const int d = i % kKtDescs;
      if (lane == 0) {
        ok = kv8_wait(&dempty[d], ((i / kKtDescs) & 1) ^ 1);
        if (ok) {
          const bool starts = from == 0, ends = to == k.nblk;
          KtDesc& D = descs[d];
          D.q0 = r.q0; D.h = h; D.r0 = k.r0; D.nr = k.nr; D.L = r.L; D.n = r.n; D.lo = k.lo; D.kend = k.kend;
          D.blk = k.blk0 + from; D.nb = to - from;
          D.slot = starts && ends ? -1 : starts ? 2 * (int)blockIdx.x + 1 : 2 * (int)blockIdx.x;
          const int parts = starts && !ends ? kv8_cta_of(pl, s0 + kKtCost + k.nblk - 1) - (int)blockIdx.x + 1 : 0;
          if (parts > 0) {  // (the run's last segment)
            Kv8Part& hd = scratch.head[blockIdx.x];
            hd.q0 = r.q0; hd.r0 = k.r0; hd.nr = k.nr; hd.h = h; hd.parts = parts;
          }
          mbar_arrive(&dfull[d]);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      // the blocks' pages' slots, a batch of `mine` blocks ahead
      const int page0 = (k.blk0 + from) * gpb, pages_end = k.kend > k.lo ? (k.kend - 1) / page + 1 : 0;
      auto look_up = [&](int j) {
        const int g = page0 + j * gpb + lane;
        return g < pages_end && j + lane / gpb < to - from ? p.page_table[(int64_t)r.row * p.pt_stride + (int64_t)g * page] : -1;
      };
      int next = look_up(0), page_slots = -1;
#pragma unroll 1
      for (int j = 0; j < to - from; ++j) {
        if (j % mine == 0) {
          page_slots = next;
          if (page0 + j * gpb + lane < pages_end && j + lane / gpb < to - from) page_slots = kv8_checked(p, page_slots);
          if (j + mine < to - from) next = look_up(j + mine);
        }
        const uint32_t x = seq + j, stage = x % C::kRaw;
        ok = kv8_wait_warp(&rempty[stage], ((x / C::kRaw) & 1) ^ 1);
        if (!ok) {
          seq = x;
          break;
        }
        const int pages = max(0, min(gpb, pages_end - (page0 + j * gpb)));
        kv8_copy_block<HD, 1>(p, &tc, &ts, raw + stage * C::kRawStage, raw_scales + stage * (C::kRawScales / 4), &rfull[stage], h, page_slots,
                           j % mine * gpb, pages);
      }
      if (!ok) break;
      seq += to - from;
      u = s0 + kKtCost + to;
      s0 += kKtCost + k.nblk;
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
    if (lane == 0) {
      if (ok) {
        if (kv8_wait(&dempty[i % kKtDescs], ((i / kKtDescs) & 1) ^ 1)) {
          descs[i % kKtDescs].nb = 0;
          mbar_arrive(&dfull[i % kKtDescs]);
        }
      } else {  // given up: the copies in flight land before the CTA's memory goes
        kv8_gave_up(720);
#pragma unroll 1
        for (uint32_t n = 1; n <= min(seq, (uint32_t)C::kRaw); ++n) {
          const uint32_t x = seq - n;
          kv8_wait(&rfull[x % C::kRaw], (x / C::kRaw) & 1);
        }
      }
    }
  } else if (warp <= 2) {
    // ------------------------------------------------------------------ products of one tile
    kt_fewer_regs<kKtRegsFew>();
    // Block after block through all segments: S of a block before O of the one before it, so that the softmax finds the next S
    // when it is done with one. (The whole warp goes through this, and one lane is elected to issue.)
    const int x = warp - 1;
    const uint32_t ts = tmem + C::kS + x * 128, to = tmem + C::kO + x * 128;
    const uint64_t q = smem_desc_sw128(smem_u32(smem + C::kOffQ + x * C::kQTile));
    constexpr uint32_t idesc_s = idesc_bf16_f32(128, kKv8Block), idesc_o = kt_idesc(128, HD) | kIdescBMajorMN;
    uint32_t g = 0, uses = 0, outs = 0;  // blocks, of them this tile's, its segments
    int i = 0, j = 0, nb = 0;
    bool ok = true, active = false;
    // the block whose O is due
    bool due = false, due_active = false, due_first = false, due_last = false;
#pragma unroll 1
    for (;;) {
      if (j == nb) {  // the next segment
        if (!(ok = kv8_wait_warp(&dfull[i % kKtDescs], (i / kKtDescs) & 1))) break;
        nb = __shfl_sync(0xffffffffu, descs[i % kKtDescs].nb, 0);
        active = __shfl_sync(0xffffffffu, descs[i % kKtDescs].nr, 0) > trows * x;
        j = 0;
        if (nb > 0 && !(ok = kv8_wait_warp(qfull, i & 1))) break;
        ++i;
      }
      if (nb > 0) {
        const uint32_t st = g % C::kStages;
        if (!(ok = kv8_wait_warp(&kfull[st], (g / C::kStages) & 1))) break;
        const int buf = 2 * x + (uses & 1);
        if (active) {
          if (uses >= 2 && !(ok = kv8_wait_warp(&pvdone[buf], ((uses - 2) >> 1) & 1))) break;
          tc_fence_after();
          if (elect_one()) {
            // (a descriptor's low bits are its address / 16)
            const uint64_t b = smem_desc_sw128(smem_u32(sK + st * C::kTile));
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              tc_mma_f16(ts + (uses & 1) * 64, q + (((kk >> 2) * C::kQHalf + (kk & 3) * 32) >> 4),
                         b + (((kk >> 2) * C::kHalf + (kk & 3) * 32) >> 4), idesc_s, kk > 0);
            tc_commit(&kempty[st]);
            tc_commit(&sfull[buf]);
            if (j == nb - 1) tc_commit(qempty);
          }
          ++uses;
        } else if (elect_one()) {
          mbar_arrive(&kempty[st]);
          if (j == nb - 1) mbar_arrive(qempty);
        }
        __syncwarp();
      }
      if (due) {  // of block g - 1
        const uint32_t st = (g - 1) % C::kStages;
        if (!(ok = kv8_wait_warp(&vfull[st], ((g - 1) / C::kStages) & 1))) break;
        if (due_active) {
          const uint32_t u = uses - 1 - (nb > 0 && active ? 1 : 0);
          if (due_first && outs > 0 && !(ok = kv8_wait_warp(&ofree[x], (outs - 1) & 1))) break;
          if (!(ok = kv8_wait_warp(&pfull[2 * x + (u & 1)], (u >> 1) & 1))) break;
          outs += due_first;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t b = smem_desc_sw128_mn(smem_u32(sV + st * C::kTile), C::kHalf);
#pragma unroll
            for (int kk = 0; kk < kKv8Block / 16; ++kk)
              tc_mma_f16_ts(to, ts + (u & 1) * 64 + kk * 8, b + (kk * 16 * 128 >> 4), idesc_o, !due_first || kk > 0);
            tc_commit(&vempty[st]);
            tc_commit(&pvdone[2 * x + (u & 1)]);
          }
        } else if (elect_one()) {
          mbar_arrive(&vempty[st]);
        }
        __syncwarp();
        // (the segment's entry: this one's, or the one before where a new segment has begun)
        if (due_last && elect_one()) mbar_arrive(&dempty[(i - 2) % kKtDescs]);
      }
      if (nb == 0) break;
      due = true;
      due_active = active;
      due_first = j == 0;
      due_last = ++j == nb;
      ++g;
    }
    if (!ok && lane == 0) kv8_gave_up(730);
    // no product is in flight when the CTA's memories go
    if (uses > 0) {
      kv8_wait_warp(&sfull[2 * x + ((uses - 1) & 1)], ((uses - 1) >> 1) & 1);
      kv8_wait_warp(&pvdone[2 * x + ((uses - 1) & 1)], ((uses - 1) >> 1) & 1);
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ queries
    kt_fewer_regs<kKtRegsFew>();
    bool ok = true;
    int i = 0;
#pragma unroll 1
    for (;; ++i) {
      const int d = i % kKtDescs;
      if (!(ok = kv8_wait_warp(&dfull[d], (i / kKtDescs) & 1))) break;
      const KtDesc D = descs[d];
      if (D.nb == 0) break;
      const int tiles = D.nr > trows ? 2 : 1, tok = D.q0 + kv8_token(p, D.r0);
      // into the L2 cache, while the last segment's are still in use
      if (i > 0 && lane < tiles * (HD / 64)) kt_prefetch_3d(&tq, lane % (HD / 64) * 64, D.h * G, tok + lane / (HD / 64) * tokens);
      if (i > 0 && !(ok = kv8_wait_warp(qempty, (i - 1) & 1))) break;
      if (elect_one()) {
        mbar_expect_tx(qfull, tiles * trows * HD * 2);
#pragma unroll 1
        for (int y = 0; y < tiles * (HD / 64); ++y)
          tma_load_3d(smem + C::kOffQ + y * C::kQHalf, &tq, qfull, y % (HD / 64) * 64, D.h * G, tok + y / (HD / 64) * tokens);
        mbar_arrive(&dempty[d]);
      }
      __syncwarp();
    }
    if (!ok) {  // given up: the copies in flight land before the CTA's memory goes
      if (lane == 0) kv8_gave_up(740);
      if (i > 0) kv8_wait_warp(qfull, (i - 1) & 1);
    }
  } else if (warp < kKtConv) {
    // ------------------------------------------------------------------ softmax
    kt_more_regs<kKtRegsSoft>();
    const int x = (warp - kKtSoft) >> 2, row = (warp & 3) * 32 + lane, t4 = lane & 3;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + C::kS + x * 128 + lane_base, to = tmem + C::kO + x * 128 + lane_base;
    const float qs = p.scale * kKv8Log2e;
    uint32_t g = 0, uses = 0;
    bool ok = true;
#pragma unroll 1
    for (int i = 0; ok; ++i) {
      const int d = i % kKtDescs;
      if (!(ok = kv8_wait_warp(&dfull[d], (i / kKtDescs) & 1))) break;
      const KtDesc D = descs[d];
      if (D.nb == 0) break;
      if (D.nr <= trows * x) {
        g += D.nb;
        __syncwarp();
        if (lane == 0) mbar_arrive(&dempty[d]);
        continue;
      }
      KtRows w;
      int least = INT_MAX, most = 0;  // of the warp's rows' positions
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int rr = (warp & 3) * 32 + (lane >> 2) + 8 * k;
        const bool in = rr < trows && x * trows + rr < D.nr;
        w.m[k] = -INFINITY;
        w.l[k] = 0.f;
        w.pos[k] = in ? D.L - D.n + kv8_token(p, D.r0 + x * trows + rr) : INT_MIN;
        if (in) least = min(least, w.pos[k]), most = max(most, w.pos[k]);
      }
      least = __reduce_min_sync(0xffffffffu, least);
      most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (w.pos[k] == INT_MIN) w.pos[k] = most;  // (a row that is none: as the last one)
      bool fresh = true;  // rows without an offset
#pragma unroll 1
      for (int j = 0; j < D.nb; ++j, ++g) {
        // (S first: a tile that sat out the last segments could take an earlier block's turn of the scales for its own)
        if (!(ok = kv8_wait_warp(&sfull[2 * x + (uses & 1)], (uses >> 1) & 1))) break;
        if (!(ok = kv8_wait_warp(&scfull[g % kKtSlots], (g / kKtSlots) & 1))) break;
        tc_fence_after();
        const KtScales& sc = slots[g % kKtSlots];
        const int k0 = (D.blk + j) * kKv8Block;
        // does every row of the warp see every key?
        const bool part = !(least >= k0 + kKv8Block - 1 && (p.window <= 0 || most - p.window < k0));
        bool moved = false;
        if (k0 > most || (p.window > 0 && k0 + kKv8Block - 1 <= least - p.window)) {  // no row sees a key of this block
          uint32_t none[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) none[k] = 0;
          kt_store_p(ts + (uses & 1) * 64, none);
          kt_store_p(ts + (uses & 1) * 64 + (16u << 16), none);
        } else {
          moved = kt_softmax(ts + (uses & 1) * 64, sc, w, qs, t4, k0, p.window, part, fresh);
        }
        if (fresh) fresh = __any_sync(0xffffffffu, w.m[0] == -INFINITY || w.m[1] == -INFINITY || w.m[2] == -INFINITY || w.m[3] == -INFINITY);
        if ((sc.bad[0] | sc.bad[1]) != 0) {  // a key that has no finite scale makes the rows that see it no numbers
          const KtSeen seen(w, k0, p.window, part);
          const uint64_t bad = sc.bad[0] | (uint64_t)sc.bad[1] << 32;
#pragma unroll 1
          for (int c = 0; c < kKv8Block; ++c)
            if (bad >> c & 1) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (c >= seen.first[k] && c < seen.end[k]) w.l[k] = __int_as_float(0x7fc00000);
            }
        }
        if (j > 0 && moved && __any_sync(0xffffffffu, w.alpha[0] != 1.f || w.alpha[1] != 1.f || w.alpha[2] != 1.f || w.alpha[3] != 1.f)) {
          // once O holds the blocks before
          if (!(ok = kv8_wait_warp(&pvdone[2 * x + ((uses - 1) & 1)], ((uses - 1) >> 1) & 1))) break;
          tc_fence_after();
          float f = 1.f;  // of this lane's row of O
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float y = __shfl_sync(0xffffffffu, w.alpha[k], (lane & 7) * 4);
            if (lane >> 3 == k) f = y;
          }
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(to + c * 32, v);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
            tmem_st_32x32b_x32(to + c * 32, v);
          }
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[2 * x + (uses & 1)]);
        ++uses;
      }
      if (!ok) break;
      // from here on a lane has one row
      const int rr = x * trows + row, r = D.r0 + rr, tok = kv8_token(p, r);
      const bool in = row < trows && rr < D.nr;
      float m = 0.f, l = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float lk = w.l[k];
        lk += __shfl_xor_sync(0xffffffffu, lk, 1);
        lk += __shfl_xor_sync(0xffffffffu, lk, 2);
        const float mk = __shfl_sync(0xffffffffu, w.m[k], (lane & 7) * 4);
        lk = __shfl_sync(0xffffffffu, lk, (lane & 7) * 4);
        if (lane >> 3 == k) m = mk, l = lk;
      }
      // O out of tensor memory, 32 head dims of 16 rows at a time, in the layout of S: of a row a lane has pairs of head dims,
      // which it trades within its four lanes for eight that follow one another. (Whole rows in a lane make stores that touch 32 lines.)
      if (!(ok = kv8_wait_warp(&pvdone[2 * x + ((uses - 1) & 1)], ((uses - 1) >> 1) & 1))) break;
      tc_fence_after();
      const int head = D.h * G + r - tok * G;
      const float f = D.slot < 0 ? kv8_norm(m, l, p.sinks, in ? head : 0) : 1.f;
      // the row's place in the output or the scratch
      const int64_t at = !in ? -1 : D.slot < 0 ? (int64_t)(D.q0 + tok) * p.nq + head : (int64_t)D.slot * kKtRows + rr;
#pragma unroll 1
      for (int c = 0; c < HD / 16; ++c) {  // head dims from 32 (c / 2) on, rows from 16 (c % 2) on
        uint32_t v[16];
        kt_load_o(to + c / 2 * 32 + ((uint32_t)(c & 1) << 20), v);
        tc_wait_ld();
        if (c == HD / 16 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ofree[x]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int src = 16 * (c & 1) + 8 * k + (lane >> 2);
          const float fk = __shfl_sync(0xffffffffu, f, src);
          const int64_t dst = __shfl_sync(0xffffffffu, at, src);
          const uint32_t* o = &v[2 * k];  // head dims 8 n + 2 t4 and the next: o[4 n], o[4 n + 1]
          if (D.slot < 0) {
            uint32_t y[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) y[n] = pack_bf16(__uint_as_float(o[4 * n]) * fk, __uint_as_float(o[4 * n + 1]) * fk);
#pragma unroll
            for (int n = 0; n < 4; n += 2) {
              const uint32_t got = __shfl_xor_sync(0xffffffffu, t4 & 1 ? y[n] : y[n + 1], 1);
              if (t4 & 1) y[n] = got;
              else y[n + 1] = got;
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const uint32_t got = __shfl_xor_sync(0xffffffffu, t4 & 2 ? y[n] : y[n + 2], 2);
              if (t4 & 2) y[n] = got;
              else y[n + 2] = got;
            }
            if (dst >= 0) reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.o) + dst * HD + c / 2 * 32)[t4] = make_uint4(y[0], y[1], y[2], y[3]);
          } else if (dst >= 0) {
            float2* to_scratch = reinterpret_cast<float2*>(scratch.o + dst * HD + c / 2 * 32) + t4;
#pragma unroll
            for (int n = 0; n < 4; ++n) to_scratch[4 * n] = make_float2(__uint_as_float(o[4 * n]), __uint_as_float(o[4 * n + 1]));
          }
        }
      }
      if (in && D.slot >= 0) scratch.ml[(int64_t)D.slot * kKtRows + rr] = make_float2(m, l);
      __syncwarp();
      if (lane == 0) mbar_arrive(&dempty[d]);
    }
    if (!ok) kv8_gave_up(750);
  } else {
    // ------------------------------------------------------------------ conversions
    kt_fewer_regs<kKtRegsConv>();
    const int w = warp - kKtConv, row = w * 32 + lane;
    // Codes: a warp takes 8 keys x 64 head dims at a time, 16 a lane, so that neither its loads nor its stores of 16
    // bytes meet in a bank: of every 8 lanes 4 have key k, the others key k ^ 5.
    const int part = lane & 3, key8 = (lane >> 3) ^ (lane & 4 ? 5 : 0);
    uint32_t g = 0;
    bool ok = true;
#pragma unroll 1
    for (int i = 0; ok; ++i) {
      const int d = i % kKtDescs;
      if (!(ok = kv8_wait_warp(&dfull[d], (i / kKtDescs) & 1))) break;
      const KtDesc D = descs[d];
      if (D.nb == 0) break;
#pragma unroll 1
      for (int j = 0; j < D.nb; ++j, ++g) {
        const uint32_t rs = g % C::kRaw, st = g % C::kStages, ph = (g / C::kStages) & 1;
        if (!(ok = kv8_wait_warp(&rfull[rs], (g / C::kRaw) & 1))) break;
        const int k0 = (D.blk + j) * kKv8Block;
        const bool partial = k0 < D.lo || k0 + kKv8Block > D.kend;  // some of the keys may be no positions
        const uint8_t* src = raw + rs * C::kRawStage;
        auto convert = [&](uint8_t* dst, int which, bool values) {
          // groups of 8 keys, w and w + 4 of them this warp's, and of 64 head dims
          uint4 v[2][HD / 64];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int key = (w + 4 * y) * 8 + key8;
            const int at = key + (key & ~(p.page - 1)) + which * p.page;  // row of the page's two parts
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
              v[y][c] = *reinterpret_cast<const uint4*>(src + at * HD + (HD == 128 ? ((c * 4 + part) ^ key8) << 4 : (part ^ (key8 >> 1)) << 4));
            if (partial && (k0 + key < D.lo || k0 + key >= D.kend)) {
#pragma unroll
              for (int c = 0; c < HD / 64; ++c) v[y][c] = make_uint4(0, 0, 0, 0);
            }
          }
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
              uint4 a, b;
              if (values) {
                kv8_to_half<FP8>(v[y][c].x, a.x, a.y);
                kv8_to_half<FP8>(v[y][c].y, a.z, a.w);
                kv8_to_half<FP8>(v[y][c].z, b.x, b.y);
                kv8_to_half<FP8>(v[y][c].w, b.z, b.w);
              } else {
                kv8_to_bf16<FP8>(v[y][c].x, a.x, a.y);
                kv8_to_bf16<FP8>(v[y][c].y, a.z, a.w);
                kv8_to_bf16<FP8>(v[y][c].z, b.x, b.y);
                kv8_to_bf16<FP8>(v[y][c].w, b.z, b.w);
              }
              uint8_t* o = dst + c * C::kHalf + ((w + 4 * y) * 8 + key8) * 128;
              *reinterpret_cast<uint4*>(o + (((2 * part) ^ key8) << 4)) = a;
              *reinterpret_cast<uint4*>(o + (((2 * part + 1) ^ key8) << 4)) = b;
            }
          fence_async_smem();
        };
        // keys, then values (one copy of the code)
#pragma unroll 1
        for (int y = 0; y < 2; ++y) {
          if (!(ok = kv8_wait_warp(&(y ? vempty : kempty)[st], ph ^ 1))) break;
          convert((y ? sV : sK) + st * C::kTile, order.codes ^ y, y);
          // scales: what used this slot before was over when its keys' products were
          if (y == 0 && row < kKv8Block) {  // (two whole warps)
            const float* sc = raw_scales + rs * (C::kRawScales / 4) + row + (row & ~(p.page - 1));
            const bool none = partial && (k0 + row < D.lo || k0 + row >= D.kend);
            float ks = none ? 0.f : sc[order.scales * p.page], vs = none ? 0.f : sc[(order.scales ^ 1) * p.page];
            const unsigned bad = __ballot_sync(0xffffffffu, !(fabsf(ks) < INFINITY) || !(fabsf(vs) < INFINITY));
            if (bad >> lane & 1) ks = vs = 0.f;
            KtScales& s = slots[g % kKtSlots];
            s.ks[row] = ks;
            s.vs[row] = vs;
            s.lv[row] = kv8_log_scale(vs);
            if (lane == 0) s.bad[w] = bad;
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&(y ? vfull : kfull)[st]);
            mbar_arrive(y ? &rempty[rs] : &scfull[g % kKtSlots]);
          }
        }
        if (!ok) break;
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&dempty[d]);
    }
    if (!ok) kv8_gave_up(760);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace msgl
