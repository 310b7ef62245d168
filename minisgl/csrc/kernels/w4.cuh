// Products with 4-bit weights and group scales: w[n, k] = (code - zero) * scale(row n, group of k).
//
// Packed weights (ops/w4.py lays them out once) are records of 32 rows by 128 inputs, [E][Nt][KC][bytes]:
//   2048 bytes of codes: two halves of 16 rows, of each two blocks of 64 inputs in the order of the tensor
//     core's A fragments: lane 4 g + t has 16 bytes = 4 words of a block. Word b holds, for
//     k = 64 block + 16 b + 4 t,
//       row g     codes k, k+1, k+2, k+3 in nibbles 0, 4, 2, 6
//       row g + 8 codes k, k+1, k+2, k+3 in nibbles 1, 5, 3, 7
//   per group of inputs 64 bytes of 16-bit scales, [8 g][half][row g, row g + 8]
//   per group 32 bytes of zero points, likewise (none: 8)
// Rows and inputs are padded to whole records with scales of zero. In a gated weight rows g of half i of a
// tile are gate rows 16 tile + 8 i + g, and rows g + 8 the up rows of the same outputs.
//
// This header is the streaming product for few tokens, which the weights' bytes bound. Every warp of a
// CTA takes an equal, contiguous run of the CTA's records and keeps the next two on their way into a ring
// of its own with bulk copies, issued by one lane once the warp has read the slot. (At 1 x 34816 x 5120 a
// producer warp for all rings measured 38 us, cp.async by every lane 27 us, bulk copies of 16-row records
// 25 us: what is left of an SM's issue slots beside the conversion decides.) A word of eight codes
// becomes one A fragment with two logic instructions and one exact subtraction per pair (a code c under
// the exponent of 2^-4 is the bf16 value 2^-4 + c 2^-11), the group's products go through mma.sync into fp32, and
// the group's scale multiplies the fp32 sums: nothing is rounded before the result. The sums are 2^-11 of the result
// until they are given away, so that a group's 128 products with codes of up to 15 stay in range whatever finite value
// the activations have. The inputs' order inside 16 is the same permutation on both sides, which is why no shuffle is
// needed.
// 1 x 34816 x 5120, groups of 128: 20.9 us, 4.4 TB/s, of which about 5 us are the launch, the first copies and the last
// tiles; 16 x 34816 x 5120 27 us (twice the products a record: the issue slots bound it).
#pragma once
#include <cuda_fp16.h>

#include <mutex>
#include <type_traits>

#include "api.h"
#include "common.cuh"

namespace msgl {

struct W4Tensor {
  const uint8_t* data;
  int tiles, kc, n, k;
};

inline W4Tensor w4_tensor(const MsglW4* w) { return {(const uint8_t*)w->data, w->tiles, w->kc, w->n, w->k}; }

constexpr int kW4Slots = 2;  // records of a warp's ring: 50 to 100 KB in flight per SM

template <int G, bool Z>
struct W4Record {
  static constexpr int kGroups = 128 / G;
  static constexpr int kScales = 2048;
  static constexpr int kZeros = kScales + kGroups * 64;
  static constexpr int kBytes = kZeros + (Z ? kGroups * 32 : 0);
  static constexpr int kRing = kW4Slots * kBytes;  // of one warp
};

// warps by the number of 8-token columns: as many as the registers of their sums allow
template <int NT>
constexpr int w4_warps() { return NT == 1 ? 24 : 16; }
template <int NT>
constexpr int w4_threads() { return w4_warps<NT>() * 32; }

// shared memory of the runs: rings, partial tiles, barriers
template <int NT, int G, bool Z>
constexpr int w4_run_bytes() { return w4_warps<NT>() * (W4Record<G, Z>::kRing + NT * 1024 + kW4Slots * 8) + 16; }

// bytes between the rows of the activations in shared memory: 32 more than a whole number of 128, so
// that the sixteen 8-byte reads of a half warp (four rows, four columns) fall into different banks
__host__ __device__ inline int w4_pitch(int inputs) { return inputs * 2 + 32; }

MSGL_DEVICE uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
MSGL_DEVICE uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
MSGL_DEVICE uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}

// asks for `bytes` (a multiple of 16, from a 16-byte boundary) to be brought into L2
MSGL_DEVICE void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// mbarrier operations and bulk_load on shared-memory addresses
MSGL_DEVICE bool mbar_try_wait_a(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// the same; the hardware may hold the warp for `ns`
MSGL_DEVICE bool mbar_try_wait_a(uint32_t bar, uint32_t parity, uint32_t ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(ns)
      : "memory");
  return ok != 0;
}
MSGL_DEVICE void mbar_expect_tx_a(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
MSGL_DEVICE void bulk_load_a(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

MSGL_DEVICE void mma_bf16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  if (first) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// bf16 pairs whose last bit is a code's unit: 128 + code, and 2^-4 + code 2^-11
constexpr uint32_t kW4Whole = 0x43004300u, kW4Small = 0x3d803d80u;
constexpr float kW4Unit = 2048.f;  // of a code under kW4Small, inverted

// two codes (bits 0-3 and 16-19 of v) under a base minus a zero point (base + zero in both halves), exactly
template <uint32_t BASE>
MSGL_DEVICE uint32_t codes_bf16x2(uint32_t v, uint32_t zero) {
  uint32_t c;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(c) : "r"(v), "n"(BASE));  // (v & 0x000f000f) | base
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&c), *reinterpret_cast<__nv_bfloat162*>(&zero));
  return *reinterpret_cast<const uint32_t*>(&d);
}

template <bool F>
MSGL_DEVICE float2 w4_scales(uint32_t v) {
  if constexpr (F) return __half22float2(*reinterpret_cast<__half2*>(&v));
  return make_float2(bf16_lo(v), bf16_hi(v));
}

// A wait that did not succeed at once. try_wait may hold the warp until the phase is over or 2 us have passed (looks 20
// to 40 ns apart by each of 26 warps took a third of an SM's issue slots). Bounded to a few seconds; false when they are
// over.
static __noinline__ __device__ bool w4_wait(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < 1 << 21; ++i)
    if (mbar_try_wait_a(bar, parity, 2000)) return true;
  report_error(kErrMbarTimeout, 400);
  return false;
}

// The runs of a CTA: its shared memory and how far the ring of this thread's warp has turned. F: fp16 scales.
template <int NT, int G, bool Z, bool F>
struct W4Runs {
  using R = W4Record<G, Z>;
  static constexpr int kWarps = w4_warps<NT>();
  static_assert(NT * 1024 <= R::kRing && R::kRing % 16 == 0, "a tile's sums fit into a ring");
  uint8_t* mem;
  uint32_t it = 0;    // records that the warp has read
  uint32_t runs = 0;  // runs so far: the phase of the activations' barrier
  bool ok = true;

  MSGL_DEVICE uint32_t ring(int warp) const { return smem_u32(mem) + warp * R::kRing; }
  // sums of a tile that the warp shares with earlier warps, and (in its ring, once that is read) with later ones
  MSGL_DEVICE float4* head(int warp) const { return reinterpret_cast<float4*>(mem + kWarps * R::kRing) + warp * NT * 64; }
  MSGL_DEVICE float4* tail(int warp) const { return reinterpret_cast<float4*>(mem + warp * R::kRing); }
  MSGL_DEVICE uint64_t* full(int warp) const {
    return reinterpret_cast<uint64_t*>(mem + kWarps * (R::kRing + NT * 1024)) + warp * kW4Slots;
  }

  MSGL_DEVICE uint32_t xbar() const { return smem_u32(mem + w4_run_bytes<NT, G, Z>() - 16); }

  // before the first run; a barrier must follow
  MSGL_DEVICE void init() {
    if (threadIdx.x < kWarps)
      for (int i = 0; i < kW4Slots; ++i) mbar_init(full(threadIdx.x) + i, 1);
    if (threadIdx.x == 0) mbar_init(reinterpret_cast<uint64_t*>(mem + w4_run_bytes<NT, G, Z>() - 16), 1);
    if (threadIdx.x < 32) fence_barrier_init();
  }

  // first record of warp i's run, of `total` records
  static MSGL_DEVICE int bound(int total, int i) { return total / kWarps * i + min(i, total % kWarps); }

  // Products of `ntiles` tiles (absolute number tile0 on) over records [c0, c0 + nc) of each with the nx rows
  // rows row(r), r < nx <= 32, of w.k bf16 each, which are brought to xs (pitch bytes apart, column 0 = record
  // c0's first input). emit(tile, acc) gets every tile's sums over kW4Unit, from one warp: acc[half][nt][0..3] = rows g,
  // g, g + 8, g + 8 of the half, of tokens 8 nt + 2 t, + 1, + 0, + 1. Tiles that several warps share are
  // summed through shared memory, in the order of the warps. Ends without a barrier: xs is free, the runs'
  // memory is for the next run only. SPLIT: nc is less than all of a tile's records.
  template <bool SPLIT, class Row, class Emit>
  MSGL_DEVICE void run(const W4Tensor& w, int64_t tile0, int ntiles, int c0, int nc, uint8_t* xs, int pitch, int nx,
                       Row row, Emit emit) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int total = ntiles * nc, a = bound(total, warp), b = bound(total, warp + 1);
    // the rows first: behind the weights' copies they would wait for these
    const int kn = min(nc * 128, w.k - c0 * 128), pad = nc * 128 - kn;
    if (warp == 0 && ok) {
      if (lane == 0) mbar_expect_tx_a(xbar(), nx * kn * 2);
      __syncwarp();
      if (lane < nx) bulk_load_a(smem_u32(xs) + lane * pitch, row(lane) + c0 * 128, kn * 2, xbar());
    }
    int tile = a / nc, cc = a - tile * nc;
    const uint32_t ring0 = ring(warp), bars = smem_u32(full(warp));
    const uint8_t* src = w.data + ((tile0 + tile) * w.kc + c0 + cc) * R::kBytes;  // next record to copy
    const int64_t skip = (int64_t)(w.kc - nc) * R::kBytes;
    int fc = cc;  // its number in its tile
    const auto fetch = [&](uint32_t slot, uint32_t bar) {
      if (lane == 0) {
        mbar_expect_tx_a(bar, R::kBytes);
        bulk_load_a(slot, src, R::kBytes, bar);
      }
      src += R::kBytes;
      if constexpr (SPLIT) {
        if (++fc == nc) {
          fc = 0;
          src += skip;
        }
      }
    };
    // the ring goes on where the previous run left it
    uint32_t slot = ring0 + (it % kW4Slots) * R::kBytes, bar = bars + (it % kW4Slots) * 8;
    constexpr uint32_t kOther = R::kBytes;
    static_assert(kW4Slots == 2, "the slots alternate");
    // A wait that fails is the last one: no copy is started after it, and those under way get as long to land.
    int most = ok ? b : 0;  // records up to here are fetched
    if (a < most) fetch(slot, bar);
    if (a + 1 < most) fetch(2 * ring0 + kOther - slot, 2 * bars + 8 - bar);
    // zeros behind the last input (pad is less than 128)
    for (int i = threadIdx.x; i < nx * (pad / 8); i += w4_threads<NT>())
      *reinterpret_cast<uint4*>(xs + i / (pad / 8) * pitch + kn * 2 + i % (pad / 8) * 16) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (ok && !(ok = w4_wait(xbar(), runs & 1))) {
      most = 0;
      if (a < b) w4_wait(bar, (it >> 1) & 1);
      if (a + 1 < b) w4_wait(2 * bars + 8 - bar, ((it + 1) >> 1) & 1);
    }
    ++runs;

    uint32_t xrow[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      xrow[nt] = smem_u32(xs) + (uint32_t)(min(nt * 8 + g, nx - 1) * pitch + t * 8);
    const uint32_t mine = lane * 16, side = R::kScales + g * 8, zside = R::kZeros + g * 4;
    float acc[2][NT][4];
    // One place gives sums away, for the size of the code: a launch of a few microseconds is mostly its first
    // execution. First the warp's own tiles, then, behind the barrier, one that it shares with later warps.
    for (int i = a;;) {
      int give = tile;
      if (i < b) {
        const int from = i - cc;            // the tile's first record
        const int end = min(from + nc, b);  // one past its last one here
        uint32_t xoff = cc * 256;
        clear(acc);
        for (; i < end; ++i) {
          if (!mbar_try_wait_a(bar, (it >> 1) & 1)) {
            if (ok && !(ok = w4_wait(bar, (it >> 1) & 1))) {
              most = 0;
              if (i + 1 < b) w4_wait(2 * bars + 8 - bar, ((it + 1) >> 1) & 1);
            }
          }
          ++it;
          uint4 q[2][2];
          uint2 s[R::kGroups];
          uint32_t z[R::kGroups];
#pragma unroll
          for (int r = 0; r < 4; ++r) q[r >> 1][r & 1] = lds128(slot + mine + r * 512);
#pragma unroll
          for (int j = 0; j < R::kGroups; ++j) {
            s[j] = lds64(slot + side + j * 64);
            if constexpr (Z) z[j] = lds32(slot + zside + j * 32);
          }
          __syncwarp();  // every lane has read the slot
          if (i + 2 < most) fetch(slot, bar);
          slot = 2 * ring0 + kOther - slot;
          bar = 2 * bars + 8 - bar;

          float tmp[2][NT][4];
#pragma unroll
          for (int quarter = 0; quarter < 4; ++quarter) {  // 32 inputs
            constexpr int per = G / 32;                    // quarters per group
            const int j = quarter / per;
            uint32_t fr[2][2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t z0 = kW4Small + (Z ? ((z[j] >> (16 * h)) & 15u) * 0x10001u : 0x00080008u);
              const uint32_t z1 = kW4Small + (Z ? ((z[j] >> (16 * h + 8)) & 15u) * 0x10001u : 0x00080008u);
              const uint4 v4 = q[h][quarter >> 1];
              const uint32_t words[2] = {quarter & 1 ? v4.z : v4.x, quarter & 1 ? v4.w : v4.y};
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                fr[h][e][0] = codes_bf16x2<kW4Small>(words[e], z0);
                fr[h][e][1] = codes_bf16x2<kW4Small>(words[e] >> 4, z1);
                fr[h][e][2] = codes_bf16x2<kW4Small>(words[e] >> 8, z0);
                fr[h][e][3] = codes_bf16x2<kW4Small>(words[e] >> 12, z1);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint2 x0 = lds64(xrow[nt] + xoff + quarter * 64), x1 = lds64(xrow[nt] + xoff + quarter * 64 + 32);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                mma_bf16_16816(tmp[h][nt], fr[h][0], x0.x, x0.y, quarter % per == 0);
                mma_bf16_16816(tmp[h][nt], fr[h][1], x1.x, x1.y, false);
              }
            }
            if (quarter % per == per - 1) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float2 sc = w4_scales<F>(h == 0 ? s[j].x : s[j].y);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  acc[h][nt][0] += tmp[h][nt][0] * sc.x;
                  acc[h][nt][1] += tmp[h][nt][1] * sc.x;
                  acc[h][nt][2] += tmp[h][nt][2] * sc.y;
                  acc[h][nt][3] += tmp[h][nt][3] * sc.y;
                }
              }
            }
          }
          xoff += 256;
        }
        cc = 0;
        ++tile;
        if (from < a || from + nc > b) {
          if (from < a) {
            put(head(warp) + lane, acc);
          } else {
            __syncwarp();
            put(tail(warp) + lane, acc);
            fence_async_smem();  // before the next run's copies
          }
          continue;
        }
      } else {
        if (i == b) __syncthreads();
        // a tile that starts in this warp's run and ends in a later warp's: sum their parts in order
        const int last = (b - 1) / nc, from = last * nc, to = from + nc;
        if (i > b || a == b || a > from || b >= to) break;
        i = b + 1;
        give = last;
        clear(acc);
        add(acc, tail(warp) + lane);
        for (int v = warp + 1; v < kWarps && bound(total, v) < min(to, total); ++v) add(acc, head(v) + lane);
      }
      emit(give, acc);
    }
  }

  static MSGL_DEVICE void clear(float (&acc)[2][NT][4]) {
#pragma unroll
    for (int i = 0; i < 8 * NT; ++i) acc[i / (4 * NT)][i / 4 % NT][i % 4] = 0.f;
  }
  // one lane's sums of a tile, 32 lanes apart
  static MSGL_DEVICE void put(float4* p, const float (&acc)[2][NT][4]) {
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      const float(&v)[4] = acc[i / NT][i % NT];
      p[i * 32] = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  static MSGL_DEVICE void add(float (&acc)[2][NT][4], const float4* p) {
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      const float4 v = p[i * 32];
      float(&o)[4] = acc[i / NT][i % NT];
      o[0] += v.x, o[1] += v.y, o[2] += v.z, o[3] += v.w;
    }
  }
};

// An activated value as the sum of two bf16 (16 bits of it): its upper half, and what is left. Infinities have nothing left.
MSGL_DEVICE void w4_act_parts(float v, __nv_bfloat16& upper, __nv_bfloat16& rest) {
  const float u = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  upper = __float2bfloat16(u);
  rest = __float2bfloat16(v == u ? 0.f : v - u);
}

// The rarer activations are a call: inlined copies would lengthen a short launch by their first execution.
static __noinline__ __device__ float w4_other_act(float g, float u, int act) {
  if (act == 1) return 0.5f * g * (1.f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g))) * u;
  // by comparison: fminf and fmaxf would drop a NaN
  g = g > 7.f ? 7.f : g;
  u = u > 7.f ? 7.f : u < -7.f ? -7.f : u;
  return g / (1.f + __expf(-1.702f * g)) * (u + 1.f);
}
MSGL_DEVICE float w4_gated_act(float g, float u, int act) {
  return act == 0 ? __fdividef(g, 1.f + __expf(-g)) * u : w4_other_act(g, u, act);
}

// kernels that a call has launched so far, and their launches
inline thread_local int w4_launched = 0;
template <typename... KArgs, typename... Args>
cudaError_t w4_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, int cluster, const Args&... args) {
  const cudaError_t e = msgl_launch(kernel, grid, block, smem, s, cluster, args...);
  if (e == cudaSuccess) ++w4_launched;
  return e;
}

// clusters of `splits` CTAs that run at once, one CTA per SM (148 SMs, in groups that are no multiples of 8)
template <auto Kernel>
int w4_resident_clusters(int splits, int threads) {
  static std::mutex mu;
  static int known[64][9] = {};
  if (splits == 1) return msgl_num_sms();
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> guard(mu);
  int& k = known[dev][splits];
  if (k != 0) return k;
  if (msgl_set_smem<Kernel>(227 * 1024) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = 227 * 1024;
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
  return k = n;
}

// calls fn(group, zeros, fp16) with the weight's form as constants
template <class Fn>
int w4_dispatch(const MsglW4* w, Fn fn) {
  const auto form = [&](auto g) {
    using std::false_type, std::true_type;
    if (w->zeros) return w->fp16 ? fn(g, true_type{}, true_type{}) : fn(g, true_type{}, false_type{});
    return w->fp16 ? fn(g, false_type{}, true_type{}) : fn(g, false_type{}, false_type{});
  };
  switch (w->group) {
    case 32: return form(std::integral_constant<int, 32>{});
    case 64: return form(std::integral_constant<int, 64>{});
    default: return form(std::integral_constant<int, 128>{});
  }
}

}  // namespace msgl
