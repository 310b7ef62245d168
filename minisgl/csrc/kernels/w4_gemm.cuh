// 4-bit products for many tokens, on the 5th-generation tensor core (layout of the weights in w4.cuh).
//
// A tile is 128 weight rows (the MMA's M) by up to 256 tokens (its N, a multiple of 16 that follows the
// number of tokens), 128 inputs per step. Roles of a CTA's 26 warps, one CTA per SM, persistent over tiles:
//   warps 0-3    epilogue, one TMEM lane quadrant each
//   warps 4-7    the tokens' rows, gathered with cp.async into a ring of 128-byte-swizzled K-major tiles
//   warp 8       bulk copies of the four records of a step into a ring of their own
//   warp 9       MMA issuer: D[128 x N] += A[128 x 128] B[N x 128]^T, fp32 in TMEM, two accumulators
//   warps 10-25  records -> bf16 A tiles: the codes become bf16 as in w4.cuh, times the group's scale
// Rounding (code - zero) * scale to bf16 is a choice: an fp32 scale applied to the sums would need the
// accumulator to be read back once per group. It adds half a step of bf16 per weight, independent from
// weight to weight, about what the result's own rounding does. The conversion bounds the kernel (11
// instructions per 8 codes, and 8 for scales and stores) up to about 128 tokens, then the tensor core.
//
// SPLIT: the CTAs of a cluster cut the inputs of one tile; each leaves its fp32 tile in its drained rings
// and sums its share of the tokens over the cluster through distributed shared memory.
#pragma once
#include "w4.cuh"

namespace msgl {

enum : int { kW4Dense = 0, kW4GateUp = 1, kW4Down = 2 };

struct W4GemmArgs {
  W4Tensor w;
  int group, zeros, fp16;
  const __nv_bfloat16* in;  // dense: [M]; gate_up: the tokens' rows; down: activated rows in sorted order
  int64_t in_stride;
  const __nv_bfloat16* bias;  // [n] of every expert
  void* out;                  // dense: bf16 [M, n]; gate_up: bf16 rows in sorted order; down: fp32 [pairs, n]
  int64_t out_stride;
  int M, bn, n_tiles, m_tiles, splits;
  // experts: tiles {expert, first sorted row, rows} of a device list, and the sorted rows' pairs
  const int* count;
  const int4* work;
  const int* sorted;
  int topk, act;
  int stages;
};

constexpr int kGwEpi = 4, kGwLoad = 4, kGwConv = 16;
constexpr int kGwThreads = (kGwEpi + kGwLoad + 2 + kGwConv) * 32;
constexpr int kGwRaw = 4 * W4Record<32, true>::kBytes, kGwRawSlots = 2;
constexpr int kGwA = 128 * 128 * 2;
constexpr int kGwMisc = 1024 + 512;  // row numbers, barriers
__host__ __device__ constexpr int w4_gemm_stage(int bn) { return kGwA + bn * 256; }
__host__ __device__ constexpr int w4_gemm_smem(int bn, int stages) {
  return 1024 + stages * w4_gemm_stage(bn) + kGwRawSlots * kGwRaw + kGwMisc;
}

MSGL_DEVICE float w4_gated_act(float g, float u, int act) {
  if (act == 0) return g / (1.f + __expf(-g)) * u;
  if (act == 1) return 0.5f * g * (1.f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g))) * u;
  g = fminf(g, 7.f);
  u = fminf(fmaxf(u, -7.f), 7.f);
  return g / (1.f + __expf(-1.702f * g)) * (u + 1.f);
}

// pair of exact integers (bf16x2) times a scale, rounded once
MSGL_DEVICE uint32_t w4_times(uint32_t v, uint32_t scale2, float scale, bool fp16) {
  if (fp16) return pack_bf16(bf16_lo(v) * scale, bf16_hi(v) * scale);
  const __nv_bfloat162 p = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<__nv_bfloat162*>(&scale2));
  return *reinterpret_cast<const uint32_t*>(&p);
}

template <int MODE, bool SPLIT>
__global__ void __launch_bounds__(kGwThreads, 1) w4_gemm_kernel(const __grid_constant__ W4GemmArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int S = p.stages, stage_bytes = w4_gemm_stage(p.bn);
  uint8_t* raw = smem + S * stage_bytes;
  int* rows = reinterpret_cast<int*>(raw + kGwRawSlots * kGwRaw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(rows + 256);
  uint64_t *raw_full = bars, *raw_empty = bars + kGwRawSlots, *a_full = raw_empty + kGwRawSlots, *b_full = a_full + 4,
           *ab_empty = b_full + 4, *tfull = ab_empty + 4, *tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = SPLIT ? (int)cluster_ctarank() : 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kGwRawSlots; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kGwConv);
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(&a_full[i], kGwConv);
      mbar_init(&b_full[i], kGwLoad);
      mbar_init(&ab_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kGwEpi);
    }
    fence_barrier_init();
  }
  const int acc_cols = p.bn <= 32 ? 32 : p.bn <= 64 ? 64 : p.bn <= 128 ? 128 : 256;
  if (warp == 9) {
    tmem_alloc(tmem_slot, 2 * acc_cols);
    tmem_relinquish();
  }
  pdl_launch();
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

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

  bool ok = true;
  if (warp < kGwEpi) {
    // ------------------------------------------------------------------ epilogue
    int use = 0;
    for (int u = u_first; u < units && ok && !SPLIT; u += u_step, ++use) {
      const Tile tl = tile_of(u);
      const int acc = use & 1;
      if (!(ok = mbar_wait(&tfull[acc], (use >> 1) & 1, 410))) break;
      tc_fence_after();
      const uint32_t d = tmem + acc * acc_cols + ((uint32_t)(warp * 32) << 16);
      const __nv_bfloat16* bias = p.bias == nullptr ? nullptr : p.bias + (int64_t)tl.e * p.w.n;
      for (int c0 = 0; c0 < tl.cols; c0 += 16) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(d + c0, r);
        tc_wait_ld();
        const int cn = min(16, tl.n - c0);
        if constexpr (MODE == kW4GateUp) {
          // even rows are gates, odd rows their ups: even lanes finish even tokens, odd lanes odd ones
          const int inter = p.w.n / 2, i = tl.nt * 64 + warp * 16 + (lane >> 1), odd = lane & 1;
          const float bg = bias != nullptr && i < inter ? __bfloat162float(bias[i]) : 0.f;
          const float bu = bias != nullptr && i < inter ? __bfloat162float(bias[inter + i]) : 0.f;
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            const float v0 = __uint_as_float(r[c]), v1 = __uint_as_float(r[c + 1]);
            const float got = __shfl_xor_sync(0xffffffffu, odd ? v0 : v1, 1);
            const float gate = odd ? got : v0, up = odd ? v1 : got;
            if (c + odd < cn && i < inter)
              reinterpret_cast<__nv_bfloat16*>(p.out)[(int64_t)(tl.row0 + c0 + c + odd) * p.out_stride + i] =
                  __float2bfloat16(w4_gated_act(gate + bg, up + bu, p.act));
          }
        } else {
          const int n = tl.nt * 128 + warp * 32 + lane;
          if (n < p.w.n) {
            const float b = bias == nullptr ? 0.f : __bfloat162float(bias[n]);
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              if (c >= cn) break;
              const float v = __uint_as_float(r[c]) + b;
              if constexpr (MODE == kW4Dense)
                reinterpret_cast<__nv_bfloat16*>(p.out)[(int64_t)(tl.row0 + c0 + c) * p.out_stride + n] = __float2bfloat16(v);
              else
                reinterpret_cast<float*>(p.out)[(int64_t)p.sorted[tl.row0 + c0 + c] * p.out_stride + n] = v;
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
    if constexpr (SPLIT) {
      // one tile per cluster: leave it as fp32 [token][128 rows] in the drained rings
      const Tile tl = tile_of(u_first);
      if (ok) ok = mbar_wait(&tfull[0], 0, 411);
      tc_fence_after();
      float* dump = reinterpret_cast<float*>(smem);
      for (int c0 = 0; c0 < tl.cols; c0 += 16) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(tmem + ((uint32_t)(warp * 32) << 16) + c0, r);
        tc_wait_ld();
#pragma unroll
        for (int c = 0; c < 16; ++c) dump[(c0 + c) * 128 + warp * 32 + lane] = __uint_as_float(r[c]);
      }
      tc_fence_before();
    }
  } else if (warp < kGwEpi + kGwLoad) {
    // ------------------------------------------------------------------ tokens' rows
    const int lt = threadIdx.x - kGwEpi * 32, chunk = lt & 15, r0 = lt >> 4;
    int stage = 0;
    uint32_t phase = 0;
    int before = -1;  // stage of the previous step, whose copies have not been waited for
    for (int u = u_first; u < units && ok; u += u_step) {
      const Tile tl = tile_of(u);
      if constexpr (MODE == kW4GateUp) {
        named_bar_sync(1, kGwLoad * 32);  // the previous tile's numbers are no longer needed
        for (int r = lt; r < tl.cols; r += kGwLoad * 32) rows[r] = p.sorted[tl.row0 + min(r, tl.n - 1)] / p.topk;
        named_bar_sync(1, kGwLoad * 32);
      }
      for (int kb = k0; kb < k1; ++kb) {
        if (!(ok = mbar_wait(&ab_empty[stage], phase ^ 1, 412))) break;
        const uint32_t dst = smem_u32(smem + stage * stage_bytes + kGwA) + (chunk >> 3) * tl.cols * 128;
        const int k = kb * 128 + chunk * 8;
        const uint32_t bytes = k < p.w.k ? 16 : 0;  // zeros beyond the last input
        const int kk = min(k, p.w.k - 8);
        for (int r = r0; r < tl.cols; r += kGwLoad * 2) {
          const int row = MODE == kW4GateUp ? rows[r] : tl.row0 + min(r, tl.n - 1);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                           dst + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)),
                       "l"(p.in + (int64_t)row * p.in_stride + kk), "r"(bytes)
                       : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (before >= 0) {
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&b_full[before]);
        }
        before = stage;
        if (++stage == S) stage = 0, phase ^= 1;
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (before >= 0) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b_full[before]);
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------------ records
    const int bytes = W4Record<128, false>::kScales + 128 / p.group * (p.zeros ? 96 : 64);
    if (lane == 0) {
      int slot = 0;
      uint32_t phase = 0;
      for (int u = u_first; u < units && ok; u += u_step) {
        const Tile tl = tile_of(u);
        const int n = min(4, p.w.tiles - tl.nt * 4);
        const uint8_t* src = p.w.data + ((int64_t)tl.e * p.w.tiles + tl.nt * 4) * p.w.kc * bytes;
        for (int kb = k0; kb < k1; ++kb) {
          if (!(ok = mbar_wait(&raw_empty[slot], phase ^ 1, 413))) break;
          mbar_expect_tx(&raw_full[slot], n * bytes);
          for (int i = 0; i < n; ++i)
            bulk_load(raw + slot * kGwRaw + i * bytes, src + ((int64_t)i * p.w.kc + kb) * bytes, bytes, &raw_full[slot]);
          if (++slot == kGwRawSlots) slot = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA
    if (lane == 0) {
      int stage = 0, use = 0;
      uint32_t phase = 0;
      for (int u = u_first; u < units && ok; u += u_step, ++use) {
        const Tile tl = tile_of(u);
        const uint32_t idesc = idesc_bf16_f32(128, tl.cols), d = tmem + (use & 1) * acc_cols;
        if (!(ok = mbar_wait(&tempty[use & 1], ((use >> 1) & 1) ^ 1, 414))) break;
        tc_fence_after();
        for (int kb = k0; kb < k1; ++kb) {
          if (!(ok = mbar_wait(&b_full[stage], phase, 415) && mbar_wait(&a_full[stage], phase, 416))) break;
          tc_fence_after();
          const uint32_t a = smem_u32(smem + stage * stage_bytes), b = a + kGwA;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            tc_mma_f16(d, smem_desc_sw128(a + (j >> 2) * (128 * 128) + (j & 3) * 32),
                       smem_desc_sw128(b + (j >> 2) * tl.cols * 128 + (j & 3) * 32), idesc, kb > k0 || j > 0);
          tc_commit(&ab_empty[stage]);
          if (++stage == S) stage = 0, phase ^= 1;
        }
        tc_commit(&tfull[use & 1]);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ records -> A tile
    // a warp's part of a step: 16 rows by 64 inputs of one record
    const int cw = warp - kGwEpi - kGwLoad - 2, ti = cw >> 2, half = (cw >> 1) & 1, block = cw & 1;
    const int g = lane >> 2, t = lane & 3;
    const int bytes = W4Record<128, false>::kScales + 128 / p.group * (p.zeros ? 96 : 64);
    const int shift = p.group == 32 ? 0 : p.group == 64 ? 1 : 2;  // quarters of a record per group
    const int zoff = W4Record<128, false>::kScales + 128 / p.group * 64;
    // rows of the A tile: as in the records, or (gated) gate and up rows in turn
    const int ra = MODE == kW4GateUp ? 2 * (ti * 16 + half * 8 + g) : ti * 32 + half * 16 + g;
    const int rb = MODE == kW4GateUp ? ra + 1 : ra + 8;
    int stage = 0, slot = 0;
    uint32_t phase = 0, rphase = 0;
    for (int u = u_first; u < units && ok; u += u_step) {
      const Tile tl = tile_of(u);
      const bool there = tl.nt * 4 + ti < p.w.tiles;
      for (int kb = k0; kb < k1; ++kb) {
        if (!(ok = mbar_wait(&raw_full[slot], rphase, 417))) break;
        const uint32_t rec = smem_u32(raw + slot * kGwRaw) + ti * bytes;
        uint4 q = make_uint4(0, 0, 0, 0);
        uint32_t s[2] = {0, 0}, z[2] = {0x0808, 0x0808};
        if (there) {
          q = lds128(rec + (half * 2 + block) * 512 + lane * 16);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int grp = (block * 2 + h) >> shift;
            s[h] = lds32(rec + W4Record<128, false>::kScales + grp * 64 + g * 8 + half * 4);
            if (p.zeros) z[h] = lds32(rec + zoff + grp * 32 + g * 4) >> (16 * half);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&raw_empty[slot]);
        if (++slot == kGwRawSlots) slot = 0, rphase ^= 1;
        if (!(ok = mbar_wait(&ab_empty[stage], phase ^ 1, 418))) break;
        if (there) {
          uint8_t* sub = smem + stage * stage_bytes + block * (128 * 128);
          const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            // neighbouring rows start with different halves of their 128 bytes: the stores of a quarter
            // warp (two rows, four chunks) then fall into different banks
            const int h = hh ^ (g & 1);
            const uint32_t w0 = h ? words[2] : words[0], w1 = h ? words[3] : words[1];
            const uint32_t sv = h ? s[1] : s[0], zv = h ? z[1] : z[0];
            const uint32_t z0 = 0x43004300u + (zv & 15u) * 0x10001u, z1 = 0x43004300u + ((zv >> 8) & 15u) * 0x10001u;
            const uint32_t sa2 = (sv & 0xffffu) * 0x10001u, sb2 = (sv >> 16) * 0x10001u;
            float2 sf = make_float2(0.f, 0.f);
            if (p.fp16) sf = w4_scales<true>(sv);
            uint32_t oa[4], ob[4];
            oa[0] = w4_times(codes_bf16x2(w0, z0), sa2, sf.x, p.fp16);
            oa[1] = w4_times(codes_bf16x2(w0 >> 8, z0), sa2, sf.x, p.fp16);
            oa[2] = w4_times(codes_bf16x2(w1, z0), sa2, sf.x, p.fp16);
            oa[3] = w4_times(codes_bf16x2(w1 >> 8, z0), sa2, sf.x, p.fp16);
            ob[0] = w4_times(codes_bf16x2(w0 >> 4, z1), sb2, sf.y, p.fp16);
            ob[1] = w4_times(codes_bf16x2(w0 >> 12, z1), sb2, sf.y, p.fp16);
            ob[2] = w4_times(codes_bf16x2(w1 >> 4, z1), sb2, sf.y, p.fp16);
            ob[3] = w4_times(codes_bf16x2(w1 >> 12, z1), sb2, sf.y, p.fp16);
            *reinterpret_cast<uint4*>(sub + ra * 128 + (((4 * h + t) ^ (ra & 7)) << 4)) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
            *reinterpret_cast<uint4*>(sub + rb * 128 + (((4 * h + t) ^ (rb & 7)) << 4)) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&a_full[stage]);
        if (++stage == S) stage = 0, phase ^= 1;
      }
    }
  }

  if constexpr (SPLIT) {
    __syncwarp();
    cluster_sync();
    // this CTA's share of the tokens: a warp per token, four rows a lane
    const Tile tl = tile_of(u_first);
    const int n = tl.nt * 128 + lane * 4;
    const int from = tl.n * rank / p.splits, to = tl.n * (rank + 1) / p.splits;
    for (int c = from + warp; c < to; c += kGwThreads / 32) {
      float v[4] = {};
      const uint32_t at = smem_u32(smem) + (c * 128 + lane * 4) * 4;
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
    tmem_dealloc(tmem, 2 * acc_cols);
  }
}

template <int MODE, bool SPLIT>
int w4_gemm_launch(W4GemmArgs p, int grid, cudaStream_t s) {
  constexpr auto kernel = w4_gemm_kernel<MODE, SPLIT>;
  constexpr int kMax = 227 * 1024;
  if (msgl_set_smem<kernel>(kMax) != cudaSuccess) return 4;
  p.stages = std::min(4, (kMax - w4_gemm_smem(p.bn, 0)) / w4_gemm_stage(p.bn));
  return msgl_launch(kernel, dim3(grid), dim3(kGwThreads), w4_gemm_smem(p.bn, p.stages), s, SPLIT ? p.splits : 1, p) ==
                 cudaSuccess
             ? 0
             : 4;
}

}  // namespace msgl
