// 4-bit products for many tokens, on the 5th-generation tensor core (layout of the weights in w4.cuh).
//
// A tile is 128 H weight rows (H = 1 or 2 MMAs of M = 128) by up to 208 tokens (their N, a multiple of 16
// that follows the number of tokens), 64 inputs per step. Roles of a CTA's 26 warps, one CTA per SM,
// persistent over tiles:
//   warps 0-3    epilogue, one TMEM lane quadrant each
//   warps 4-7    the tokens' rows into a ring of 128-byte-swizzled K-major tiles: one TMA copy per step (dense),
//                one per 16 rows (down), or gathered by token with cp.async (gate_up)
//   warp 8       bulk copies of the tile's records of 128 inputs (two steps) into a ring of their own
//   warp 9       MMA issuer: D_h[128 x N] += A_h[128 x 64] B[N x 64]^T, fp32 in TMEM, two sets if they fit
//   warps 10-25  records -> bf16 A tiles in tensor memory: the codes become bf16 as in w4.cuh, times the group's
//                scale (experts: its two parts). Half of them take the even steps, half the odd ones: one half
//                converts while the other waits for its barriers and its stores.
// What bounds it is the conversion's issue slots (about 1000 warp instructions of a step's 1900; 64% of the slots are used
// at 32 tokens, the tensor pipe 17% of the time) and, next to it, the latency of one step through conversion, MMA and
// release: 640 clocks a step with few tokens, 17 x 34816 x 5120 33 us; 200 x 34816 x 5120 57 us, 1.26 PFLOP/s, 75% of a
// measured bf16 product's rate; 1024 tokens 271 to 276 us, 79%. fp16 scales are multiplied in fp32 and cost more: 64
// tokens 46 us (bf16 37), 200 tokens 65 (56), 1024 tokens 363 (271); zero points 1 to 8% with either.
// A comes from tensor memory because shared memory's 128 bytes a clock were the limit with A tiles there
// (200 tokens: 143 KB a step, of which A written and read 64): 72 us at 200 x 34816 x 5120.
// Rounding (code - zero) * scale to bf16 is a choice of the dense product: an fp32 scale applied to the sums would need
// the accumulator to be read back once per group. It adds half a step of bf16 per weight, independent from weight to
// weight, about what the result's own rounding does: 0.0022 off in the 2-norm where exact weights give 0.0017.
// The experts' two products in a row would be 0.0033 to 0.0037 off. Their weights are exact: a scale is the sum of its
// first four bits and the rest, a code times the first is exact in bf16, times the rest too (fp16 scales leave 7 bits: off
// by half a step of bf16 of an eighth of the weight at most, 2^-12 of it), and both are tiles of A, multiplied one after
// the other into the same sums: 0.0023, which is what the roundings of the activated values and of the result leave. The
// price, 128 experts of 2048 x 768, 8 a token, beside rounded weights: 512 tokens 181 us and 160, 2048 tokens 400 and
// 334; with fp16 scales 512 tokens 190 and 192.
//
// 256 rows per tile (H = 2) because the tokens' rows come from L2 once per tile: with 128 rows 200 tokens x
// 34816 x 5120 read 560 MB of them, 145 us. H = 1 where 256-row tiles would leave SMs idle.
//
// SPLIT: the CTAs of a cluster cut the inputs of one tile; each leaves its fp32 tile in its drained rings
// and sums its share of the tokens over the cluster through distributed shared memory.
#pragma once
#include <mutex>

#include "w4.cuh"

namespace msgl {

enum : int { kW4Dense = 0, kW4GateUp = 1, kW4Down = 2 };

struct W4GemmArgs {
  W4Tensor w;
  int group, zeros, fp16;
  const __nv_bfloat16* in;  // dense: [M]; gate_up: the tokens' rows; down: activated rows in sorted order
  int64_t in_stride;
  const __nv_bfloat16* bias;  // [n] of every expert
  void* out;                  // dense: bf16 [M, n]; gate_up: bf16, down: fp32 rows in sorted order
  int64_t out_stride;
  int M, bn, n_tiles, m_tiles, splits;
  // experts: tiles {expert, first sorted row, rows} of a device list, and the sorted rows' pairs
  const int* count;
  const int4* work;
  const int* sorted;
  int topk, act;
  int sets, half_cols;           // accumulators: sets of H x half_cols columns
  int stages, slots, raw_bytes;  // rings: A, records of two steps
  int ring_bytes;                // all of them, or the fp32 tile if that is larger
};

constexpr int kGwEpi = 4, kGwLoad = 4, kGwConv = 16;
constexpr int kGwThreads = (kGwEpi + kGwLoad + 2 + kGwConv) * 32;
constexpr int kGwMaxSlots = 8, kGwMaxA = 8;  // most stages of the rings
constexpr int kGwMaxB = 8;
constexpr int w4_row_stages(int mode) { return mode == kW4GateUp ? kGwMaxB : 4; }  // of the tokens' rows
// A tiles that a weight is given as. One: (code - zero) * scale rounded to bf16. Two: the products with the scale's
// first four bits, which are exact in bf16, and with the rest of it, which are exact for bf16 scales.
constexpr int w4_parts(int mode) { return mode == kW4Dense ? 1 : 2; }
constexpr int kGwMaxGather = 128;  // gathered tokens of a tile
constexpr int kGwMisc = kGwLoad * kGwMaxGather * 4 + 512;  // row numbers, barriers
constexpr int kGwRoom = 227 * 1024 - 1024 - kGwMisc;  // of the rings
constexpr int kGwMaxTokens = 208;    // of a tile: three half-step stages of A then fit beside the accumulators

// pair of exact integers (bf16x2) times a scale, rounded once
template <bool F>
MSGL_DEVICE uint32_t w4_times(uint32_t v, uint32_t scale2, float scale) {
  if constexpr (F) return pack_bf16(bf16_lo(v) * scale, bf16_hi(v) * scale);
  const __nv_bfloat162 p = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<__nv_bfloat162*>(&scale2));
  return *reinterpret_cast<const uint32_t*>(&p);
}

// two scales as bf16 pairs that sum to them: their first four bits (the leading one among them), and the rest
template <bool F>
MSGL_DEVICE void w4_scale_parts(uint32_t scales, uint32_t (&part)[2]) {
  if constexpr (F) {
    uint32_t top = scales & 0xff80ff80u;
    const __half2 rest = __hsub2(*reinterpret_cast<__half2*>(&scales), *reinterpret_cast<__half2*>(&top));
    const float2 t = w4_scales<true>(top), r = __half22float2(rest);
    part[0] = pack_bf16(t.x, t.y);
    part[1] = pack_bf16(r.x, r.y);
  } else {
    part[0] = scales & 0xfff0fff0u;
    const __nv_bfloat162 rest = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&scales), *reinterpret_cast<__nv_bfloat162*>(&part[0]));
    part[1] = *reinterpret_cast<const uint32_t*>(&rest);
  }
}

// 16 lanes x 16 columns of tensor memory from the warp's registers: r[4i], r[4i + 1] are columns 8i + 2t,
// 8i + 2t + 1 of lane g, r[4i + 2], r[4i + 3] those of lane g + 8 (thread 4 g + t)
MSGL_DEVICE void tmem_st_16x256b_x2(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// 16 bytes, or zeros if `bytes` is 0
MSGL_DEVICE void cp_async_zfill(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// a role's wait: true once the phase is complete, false if it never is
MSGL_DEVICE bool w4_await(uint64_t* bar, uint32_t parity) {
  const uint32_t a = smem_u32(bar);
  return mbar_try_wait_a(a, parity) || w4_wait(a, parity);
}

template <int MODE, int H, bool SPLIT, bool FINE, bool Z, bool F>
__global__ void __launch_bounds__(kGwThreads, 1)
w4_gemm_kernel(const __grid_constant__ W4GemmArgs p, const __grid_constant__ CUtensorMap rows_map) {
  static_assert(MODE != kW4GateUp || H == 2, "gate rows in one half, up rows in the other");
  constexpr int kRecs = 4 * H, kGwB = w4_row_stages(MODE);
  // Columns of a half in a stage of A, by parts. FINE: a stage is half a step, so that three fit beside the accumulators of
  // more than 192 tokens; the MMA warp then waits and commits twice a step, which small tiles would feel. (One issue
  // of a step's eight MMAs against two of four: 17 tokens 34.4 and 35.8 us, 256 tokens 87.8 and 84.7.)
  constexpr int kPart = FINE ? 16 : 32, kCols = kPart * w4_parts(MODE);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = p.stages, stage_bytes = p.bn * 128;
  uint8_t* raw = smem + kGwB * stage_bytes;
  int* rows = reinterpret_cast<int*>(smem + p.ring_bytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(rows + kGwLoad * kGwMaxGather);
  uint64_t *raw_full = bars, *raw_empty = bars + kGwMaxSlots, *a_full = raw_empty + kGwMaxSlots,
           *a_empty = a_full + kGwMaxA, *b_full = a_empty + kGwMaxA, *b_empty = b_full + kGwMaxB, *tfull = b_empty + kGwMaxB,
           *tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = SPLIT ? (int)cluster_ctarank() : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.slots; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kGwConv);
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(&a_full[i], kGwConv / 2);
      mbar_init(&a_empty[i], 1);
    }
    for (int i = 0; i < kGwB; ++i) {
      mbar_init(&b_full[i], 1);
      mbar_init(&b_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kGwEpi);
    }
    fence_barrier_init();
    if constexpr (MODE != kW4GateUp) prefetch_tmap(&rows_map);
  }
  // tensor memory: accumulators from column 0, A stages of H x kCols columns at the end
  const int sets = p.sets, half_cols = p.half_cols;
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_launch();
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all of tensor memory was allocated, so it begins at column 0
  constexpr uint32_t tmem = 0;
  const uint32_t tmem_a = 512 - S * H * kCols;
  if (*tmem_slot != 0 && threadIdx.x == 0) report_error(kErrBounds, 420);

  const int units = p.n_tiles * (MODE == kW4Dense ? p.m_tiles : *p.count);
  const int u_first = SPLIT ? blockIdx.x / p.splits : blockIdx.x, u_step = SPLIT ? units : gridDim.x;
  const int k0 = SPLIT ? p.w.kc * rank / p.splits : 0, k1 = SPLIT ? p.w.kc * (rank + 1) / p.splits : p.w.kc;
  // a tile: expert, weight tile, first token (sorted) row, rows, and the MMA's N
  struct Tile {
    int e, nt, row0, n, cols;
  };
  const auto tile_of = [&](int u) {
    Tile t;
    const int mt = u / p.n_tiles;
    t.nt = u - mt * p.n_tiles;
    if constexpr (MODE == kW4Dense) {
      t.e = 0;
      t.row0 = mt * p.bn;
      t.n = min(p.bn, p.M - t.row0);
    } else {
      const int4 wk = p.work[mt];
      t.e = wk.x;
      t.row0 = wk.y;
      t.n = wk.z;
    }
    t.cols = (t.n + 15) & ~15;
    return t;
  };
  // set and phase of the n-th tile of this CTA
  const auto set_of = [&](int n) { return sets == 2 ? n & 1 : 0; };
  const auto set_phase = [&](int n) { return (uint32_t)(sets == 2 ? n >> 1 : n) & 1; };

  bool ok = true;
  if (warp < kGwEpi) {
    // ------------------------------------------------------------------ epilogue
    int use = 0;
    for (int u = u_first; u < units && ok && !SPLIT; u += u_step, ++use) {
      const Tile tl = tile_of(u);
      const int set = set_of(use);
      if (!(ok = w4_await(&tfull[set], set_phase(use)))) break;
      tc_fence_after();
      const uint32_t d = tmem + set * H * half_cols + ((uint32_t)(warp * 32) << 16);
      const __nv_bfloat16* bias = p.bias == nullptr ? nullptr : p.bias + (int64_t)tl.e * p.w.n;
      for (int c0 = 0; c0 < tl.cols; c0 += 16) {
        const int cn = min(16, tl.n - c0);
        uint32_t r[H][16];
#pragma unroll
        for (int h = 0; h < H; ++h) tmem_ld_32x32b_x16(d + h * half_cols + c0, r[h]);
        tc_wait_ld();
        if constexpr (MODE == kW4GateUp) {
          const int inter = p.w.n / 2, i = tl.nt * 128 + warp * 32 + lane;
          const float bg = bias != nullptr && i < inter ? __bfloat162float(bias[i]) : 0.f;
          const float bu = bias != nullptr && i < inter ? __bfloat162float(bias[inter + i]) : 0.f;
          float v[16];
          if (p.act == 0) {
#pragma unroll
            for (int c = 0; c < 16; ++c) v[c] = w4_gated_act(__uint_as_float(r[0][c]) + bg, __uint_as_float(r[H - 1][c]) + bu, 0);
          } else {
#pragma unroll
            for (int c = 0; c < 16; ++c)
              v[c] = w4_other_act(__uint_as_float(r[0][c]) + bg, __uint_as_float(r[H - 1][c]) + bu, p.act);
          }
          __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.out) + (int64_t)(tl.row0 + c0) * p.out_stride + i;
#pragma unroll
          for (int c = 0; c < 16; ++c, o += p.out_stride)
            if (c < cn && i < inter) *o = __float2bfloat16(v[c]);
        } else {
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const int n = (tl.nt * H + h) * 128 + warp * 32 + lane;
            const float b = bias == nullptr || n >= p.w.n ? 0.f : __bfloat162float(bias[n]);
            if (n >= p.w.n) continue;
            using Out = std::conditional_t<MODE == kW4Dense, __nv_bfloat16, float>;
            Out* o = reinterpret_cast<Out*>(p.out) + (int64_t)(tl.row0 + c0) * p.out_stride + n;
#pragma unroll
            for (int c = 0; c < 16; ++c, o += p.out_stride)
              if (c < cn) *o = Out(__uint_as_float(r[h][c]) + b);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[set]);
    }
    if constexpr (SPLIT) {
      // one tile per cluster: leave it as fp32 [token][128 H rows] in the drained rings
      const Tile tl = tile_of(u_first);
      if (ok) ok = w4_await(&tfull[0], 0);
      tc_fence_after();
      float* dump = reinterpret_cast<float*>(smem);
      for (int c0 = 0; c0 < tl.cols; c0 += 16)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(tmem + ((uint32_t)(warp * 32) << 16) + h * half_cols + c0, r);
          tc_wait_ld();
#pragma unroll
          for (int c = 0; c < 16; ++c) dump[((c0 + c) * H + h) * 128 + warp * 32 + lane] = __uint_as_float(r[c]);
        }
      tc_fence_before();
    }
  } else if (warp < kGwEpi + kGwLoad) {
    // ------------------------------------------------------------------ tokens' rows
    int stage = 0;
    uint32_t phase = 0;
    if constexpr (MODE != kW4GateUp) {
      if (warp == kGwEpi && lane == 0) {
        for (int u = u_first; u < units && ok; u += u_step) {
          const Tile tl = tile_of(u);
          for (int ks = 2 * k0; ks < 2 * k1; ++ks) {
            if (!(ok = w4_await(&b_empty[stage], phase ^ 1))) break;
            uint8_t* dst = smem + stage * stage_bytes;
            // rows beyond the last one and inputs beyond the last one arrive as zeros, and count
            if constexpr (MODE == kW4Dense) {
              mbar_expect_tx(&b_full[stage], p.bn * 128);
              tma_load_2d(dst, &rows_map, &b_full[stage], ks * 64, tl.row0);
            } else {
              mbar_expect_tx(&b_full[stage], tl.cols * 128);
              for (int r = 0; r < tl.cols; r += 16) tma_load_2d(dst + r * 128, &rows_map, &b_full[stage], ks * 64, tl.row0 + r);
            }
            if (++stage == kGwB) stage = 0, phase ^= 1;
          }
        }
      }
      __syncwarp();
    } else {
      // A warp per step, in turn: a step's cost is mostly one chain of dependent instructions (four warps with a
      // quarter of every step's rows each were the products' limit).
      const int lw = warp - kGwEpi, chunk = lane & 7, r0 = lane >> 3;
      int* const mine = rows + lw * kGwMaxGather;
      const uint32_t even = r0 * 128 + ((chunk ^ r0) << 4), odd = even ^ 64;  // rows 8 i + r0, 8 i + r0 + 4 (swizzled)
      int step = 0;
      for (int u = u_first; u < units; u += u_step) {
        const Tile tl = tile_of(u);
        __syncwarp();  // the previous tile's numbers are no longer needed
        for (int r = lane; r < tl.cols; r += 32) mine[r] = p.sorted[tl.row0 + min(r, tl.n - 1)] / p.topk;
        __syncwarp();
        for (int ks = 2 * k0; ks < 2 * k1; ++ks, ++step) {
          if (step % kGwLoad != lw) continue;
          const int st = step % kGwB;
          if (ok) ok = w4_await(&b_empty[st], (step / kGwB & 1) ^ 1);
          __syncwarp();
          uint32_t dst = smem_u32(smem) + st * stage_bytes;
          const int k = ks * 64 + chunk * 8;
          const uint32_t bytes = k < p.w.k ? 16 : 0;  // zeros beyond the last input
          const __nv_bfloat16* src = p.in + min(k, p.w.k - 8);
#pragma unroll 2
          for (int r = r0; r < tl.cols; r += 8, dst += 1024) {
            cp_async_zfill(dst + even, src + (int64_t)mine[r] * p.in_stride, bytes);
            cp_async_zfill(dst + 512 + odd, src + (int64_t)mine[r + 4] * p.in_stride, bytes);
          }
          asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&b_full[st]);
        }
      }
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------------ records
    const int bytes = p.raw_bytes / kRecs;
    const uint32_t raw0 = smem_u32(raw), full0 = smem_u32(raw_full);
    int slot = 0;
    uint32_t phase = 0;
    for (int u = u_first; u < units && ok; u += u_step) {
      const Tile tl = tile_of(u);
      const int n = min(kRecs, p.w.tiles - tl.nt * kRecs);
      const uint8_t* src = p.w.data + (((int64_t)tl.e * p.w.tiles + tl.nt * kRecs) * p.w.kc + k0) * bytes;
      for (int kb = k0; kb < k1; ++kb, src += bytes) {
        if (!(ok = w4_await(&raw_empty[slot], phase ^ 1))) break;
        if (elect_one()) {
          mbar_expect_tx_a(full0 + slot * 8, n * bytes);
#pragma unroll
          for (int i = 0; i < kRecs; ++i)
            if (i < n)
              bulk_load_a(raw0 + slot * p.raw_bytes + i * bytes, src + (int64_t)i * p.w.kc * bytes, bytes, full0 + slot * 8);
        }
        __syncwarp();
        if (++slot == p.slots) slot = 0, phase ^= 1;
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA
    // The whole warp runs the loop, so that the descriptors stay in uniform registers; one lane issues. (Leaving the
    // loop on a failed wait is faster than running on without waits: 200 tokens 56.7 us and 60.7.)
    int stage = 0, bstage = 0, use = 0;
    uint32_t phase = 0, bphase = 0;
    for (int u = u_first; u < units && ok; u += u_step, ++use) {
      const Tile tl = tile_of(u);
      const uint32_t idesc = idesc_bf16_f32(128, tl.cols), d = set_of(use) * H * half_cols;
      if (!(ok = w4_await(&tempty[set_of(use)], set_phase(use) ^ 1))) break;
      tc_fence_after();
      bool acc = false;
      for (int ks = 2 * k0; ks < 2 * k1; ++ks) {
        if (!(ok = w4_await(&b_full[bstage], bphase))) break;
        const uint64_t b = smem_desc_sw128(smem_u32(smem) + bstage * stage_bytes);
#pragma unroll
        for (int e = 0; e < 2; e += FINE ? 1 : 2) {
          if (!(ok = w4_await(&a_full[stage], phase))) break;
          tc_fence_after();
          const uint32_t a = 512 - (S - stage) * H * kCols;
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < (FINE ? 2 : 4); ++j)
#pragma unroll
              for (int h = 0; h < H; ++h)
#pragma unroll
                for (int q = 0; q < w4_parts(MODE); ++q)
                  tc_mma_f16_ts(d + h * half_cols, a + h * kCols + q * kPart + j * 8, b + e * 4 + j * 2, idesc,
                                acc || e > 0 || j > 0 || q > 0);
            tc_commit(&a_empty[stage]);
            if (!FINE || e == 1) tc_commit(&b_empty[bstage]);
          }
          __syncwarp();
          if (++stage == S) stage = 0, phase ^= 1;
        }
        if (!ok) break;
        acc = true;
        if (++bstage == kGwB) bstage = 0, bphase ^= 1;
      }
      if (elect_one()) tc_commit(&tfull[set_of(use)]);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ records -> A tile
    // A warp's part of a step: 64 inputs of 16 H rows of a record (H = 1: two warps share a record). It writes
    // the 32 lanes that its number modulo 4 gives it: records go to the rows of the tile in their order, or
    // (gated) their gate rows to one half of the tile and their up rows to the other, 16 lanes each.
    const int cw = warp - kGwEpi - kGwLoad - 2, quad = warp & 3, other = cw >> 2;  // four warps of each quadrant
    const int block = other & 1, m = other >> 1;
    const int ti = MODE == kW4GateUp ? quad * 2 + m : H == 2 ? quad + 4 * m : quad;
    const int g = lane >> 2, t = lane & 3;
    const int bytes = p.raw_bytes / kRecs;
    const int shift = p.group == 32 ? 0 : p.group == 64 ? 1 : 2;  // quarters of a record per group
    const int zoff = W4Record<128, false>::kScales + 128 / p.group * 64;
    const uint32_t raw0 = smem_u32(raw);
    const uint32_t lanes = (uint32_t)(quad * 32 + (MODE == kW4GateUp ? m * 16 : 0)) << 16;
    int stage = 0, slot = 0;  // stage of the step of both halves that comes next
    uint32_t phase = 0, rphase = 0;
    const auto advance = [&](int n) {
      for (stage += n; stage >= S; stage -= S) phase ^= 1;
    };
    constexpr int kStages = FINE ? 2 : 1;  // of a step
    if (block == 1) advance(kStages);
    for (int u = u_first; u < units && ok; u += u_step) {
      for (int kb = k0; kb < k1; ++kb) {
        if (!(ok = w4_await(&raw_full[slot], rphase))) break;
        // (records behind the weight's last one are whatever the slot holds: their rows of the result are not stored)
        const uint32_t rec = raw0 + slot * p.raw_bytes + ti * bytes;
        uint4 q[H];
        uint2 s[2];
        uint32_t z[2];
#pragma unroll
        for (int i = 0; i < H; ++i) q[i] = lds128(rec + ((H == 2 ? i : m) * 2 + block) * 512 + lane * 16);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int grp = (2 * block + e) >> shift;
          s[e] = lds64(rec + W4Record<128, false>::kScales + grp * 64 + g * 8);
          z[e] = Z ? lds32(rec + zoff + grp * 32 + g * 4) : 0x08080808u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&raw_empty[slot]);
        if (++slot == p.slots) slot = 0, rphase ^= 1;
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // 32 inputs
          // a store's registers: two words by rows g (two pairs of inputs) and rows g + 8 of a half; gated: by the gate
          // rows (first store) or the up rows (second) of both halves
          uint32_t r[H][8];
          uint32_t parts[H][2][2];  // by half, part and row: a scale in both halves of a register
#pragma unroll
          for (int i = 0; i < H; ++i) {
            const int half = H == 2 ? i : m;
            const uint32_t sv = half ? s[e].y : s[e].x, zv = z[e] >> (16 * half);
            const uint32_t z0 = kW4Whole + (Z ? (zv & 15u) * 0x10001u : 0x00080008u);
            const uint32_t z1 = kW4Whole + (Z ? ((zv >> 8) & 15u) * 0x10001u : 0x00080008u);
            const uint32_t sa2 = __byte_perm(sv, 0, 0x1010), sb2 = __byte_perm(sv, 0, 0x3232);
            float2 sf = make_float2(0.f, 0.f);
            if constexpr (w4_parts(MODE) == 2) {
              uint32_t part[2];
              w4_scale_parts<F>(sv, part);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                parts[i][k][0] = __byte_perm(part[k], 0, 0x1010);
                parts[i][k][1] = __byte_perm(part[k], 0, 0x3232);
              }
            } else if constexpr (F) {
              sf = w4_scales<true>(sv);
            }
            const uint32_t words[2] = {e ? q[i].z : q[i].x, e ? q[i].w : q[i].y};
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              uint32_t* const lo = MODE == kW4GateUp ? &r[0][4 * b + 2 * i] : &r[i][4 * b];
              uint32_t* const hi = MODE == kW4GateUp ? &r[H - 1][4 * b + 2 * i] : &r[i][4 * b + 2];
              // (two parts: the codes alone, times the parts of their scales below)
              const auto value = [&](uint32_t word, uint32_t zero, uint32_t s2, float s) {
                const uint32_t v = codes_bf16x2<kW4Whole>(word, zero);
                return w4_parts(MODE) == 2 ? v : w4_times<F>(v, s2, s);
              };
              lo[0] = value(words[b], z0, sa2, sf.x);
              hi[0] = value(words[b] >> 4, z1, sb2, sf.y);
              lo[1] = value(words[b] >> 8, z0, sa2, sf.x);
              hi[1] = value(words[b] >> 12, z1, sb2, sf.y);
            }
          }
          if (FINE || e == 0) {
            if (ok) ok = w4_await(&a_empty[stage], phase ^ 1);
            if (!ok) break;
            tc_fence_after();
          }
          const uint32_t dst = tmem_a + lanes + stage * H * kCols + (FINE ? 0 : e * 16);
#pragma unroll
          for (int i = 0; i < H; ++i) {
            const uint32_t to = MODE == kW4GateUp ? dst + i * kCols
                                                  : dst + (H == 2 ? m * kCols : 0) + ((uint32_t)((H == 2 ? i : m) * 16) << 16);
            if constexpr (w4_parts(MODE) == 1) {
              tmem_st_16x256b_x2(to, r[i]);
            } else {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                uint32_t o[8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                  o[c] = w4_times<false>(r[i][c], MODE == kW4GateUp ? parts[c / 2 % 2][k][i] : parts[i][k][c / 2 % 2], 0.f);
                tmem_st_16x256b_x2(to + k * kPart, o);
              }
            }
          }
          if (FINE || e == 1) {
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&a_full[stage]);
            advance(1);
          }
        }
        if (!ok) break;
        advance(kStages);  // the other warps' step
      }
    }
  }

  if constexpr (SPLIT) {
    __syncwarp();
    cluster_sync();
    // this CTA's share of the tokens: a warp per token and 128 rows, four rows a lane
    const Tile tl = tile_of(u_first);
    const int from = tl.n * rank / p.splits, to = tl.n * (rank + 1) / p.splits;
    for (int ch = from * H + warp; ch < to * H; ch += kGwThreads / 32) {
      const int c = ch / H, n = (tl.nt * H + ch % H) * 128 + lane * 4;
      float v[4] = {};
      const uint32_t at = smem_u32(smem) + (ch * 128 + lane * 4) * 4;
      for (int r = 0; r < p.splits; ++r) {
        const float4 f = ld_dsmem_v4(dsmem_addr(at, r));
        v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
      }
      __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.out) + (int64_t)(tl.row0 + c) * p.out_stride + n;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (p.bias != nullptr && n + i < p.w.n) v[i] += __bfloat162float(p.bias[n + i]);
      if (p.out_stride % 4 == 0 && n + 3 < p.w.n) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < p.w.n) o[i] = __float2bfloat16(v[i]);
      }
    }
    cluster_sync();  // the other CTAs read this one's rings
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

typedef CUresult (*W4EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// bf16 rows [rows, cols] with boxes of 64 columns x box_rows, 128-byte swizzle; false if it cannot be encoded
inline bool w4_rows_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t stride, int box_rows) {
  static W4EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<W4EncodeFn>(ptr);
  });
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, ones,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE, int H, bool SPLIT, bool FINE, bool Z, bool F>
int w4_gemm_launch_as(W4GemmArgs p, int grid, cudaStream_t s) {
  constexpr auto kernel = w4_gemm_kernel<MODE, H, SPLIT, FINE, Z, F>;
  constexpr int kMax = 227 * 1024, kGwB = w4_row_stages(MODE);
  if (msgl_set_smem<kernel>(kMax) != cudaSuccess) return 4;
  // Tensor memory's 512 columns: two sets of accumulators if two steps of A fit beside them, else one and up to
  // eight stages. Shared memory: four stages of the tokens' rows, and up to eight steps' records (a copy
  // takes about 1 us).
  constexpr int kA = H * (FINE ? 16 : 32) * w4_parts(MODE);
  p.half_cols = p.bn;
  p.sets = 512 - 2 * H * p.half_cols >= (FINE ? 3 : 2) * kA ? 2 : 1;
  p.stages = std::min(kGwMaxA, (512 - p.sets * H * p.half_cols) / kA);
  // A team of converters waits for a stage's turn by the parity of its phase, and takes every other step: its last wait
  // must have shown that all but the latest of the stage's turns are over. That is so with two stages of a step, or
  // three of half a step.
  if (p.stages < (FINE ? 3 : 2) || (MODE == kW4GateUp && p.bn > kGwMaxGather)) return 3;
  p.raw_bytes = 4 * H * (W4Record<128, false>::kScales + 128 / p.group * (Z ? 96 : 64));
  const int room = kGwRoom, stage = p.bn * 128;
  p.slots = std::min(kGwMaxSlots, (room - kGwB * stage) / p.raw_bytes);
  p.ring_bytes = kGwB * stage + p.slots * p.raw_bytes;
  if (SPLIT) p.ring_bytes = std::max(p.ring_bytes, p.bn * H * 512);
  if (p.ring_bytes > room) return 3;
  CUtensorMap map = {};
  if (MODE != kW4GateUp &&
      !w4_rows_map(&map, p.in, p.M, p.w.k, p.M == 1 ? (int64_t)p.w.k : p.in_stride, MODE == kW4Dense ? p.bn : 16))
    return 2;
  const int smem = 1024 + kGwMisc + p.ring_bytes;
  return w4_launch(kernel, dim3(grid), dim3(kGwThreads), smem, s, SPLIT ? p.splits : 1, p, map) == cudaSuccess ? 0 : 4;
}

// clusters of s CTAs of the dense form that run at once
template <int H>
int w4_gemm_clusters(int s) { return w4_resident_clusters<w4_gemm_kernel<kW4Dense, H, true, false, false, false>>(s, kGwThreads); }

template <int MODE, int H, bool SPLIT, bool FINE>
int w4_gemm_launch_form(const W4GemmArgs& p, int grid, cudaStream_t s) {
  if (p.zeros)
    return p.fp16 ? w4_gemm_launch_as<MODE, H, SPLIT, FINE, true, true>(p, grid, s)
                  : w4_gemm_launch_as<MODE, H, SPLIT, FINE, true, false>(p, grid, s);
  return p.fp16 ? w4_gemm_launch_as<MODE, H, SPLIT, FINE, false, true>(p, grid, s)
                : w4_gemm_launch_as<MODE, H, SPLIT, FINE, false, false>(p, grid, s);
}

template <int MODE, int H, bool SPLIT>
int w4_gemm_launch(const W4GemmArgs& p, int grid, cudaStream_t s) {
  if constexpr (MODE == kW4Dense && H == 2) {
    if (p.bn > 192) return w4_gemm_launch_form<MODE, H, SPLIT, true>(p, grid, s);
  }
  return w4_gemm_launch_form<MODE, H, SPLIT, false>(p, grid, s);
}

}  // namespace msgl
