// Products with 4-bit weights and group scales: w[n, k] = (code - zero) * scale(row n, group of k).
//
// Packed weights (ops/w4.py lays them out once): tiles of 16 rows by 64 inputs, 512 bytes each, in the
// order of the tensor core's A fragments, so that a warp's 16-byte loads are one tile:
//   q [E][Nt][KB][32 lanes][4 words], lane = 4 g + t. Word 2h + j holds, for k = 64 kb + 32 h + 8 t + 4 j,
//     row g     codes k, k+1, k+2, k+3 in nibbles 0, 4, 2, 6
//     row g + 8 codes k, k+1, k+2, k+3 in nibbles 1, 5, 3, 7
//   s [E][Nt][KG][8][2] 16-bit scales of rows g and g + 8, z likewise in bytes (none: 8).
// Rows and inputs are padded to whole tiles with scales of zero. In a gated weight rows 0-7 of a tile
// are gate rows 8 i .. 8 i + 7 and rows 8-15 the up rows of the same outputs.
//
// This header is the streaming product for few tokens (the weight bytes bound it): every warp of a
// CTA takes an equal, contiguous run of the CTA's weight tiles and keeps kDepth of them in flight in
// registers; a word of eight codes becomes one A fragment with two logic instructions and one exact
// subtraction per pair (a code c under the exponent of 128 is the bf16 value 128 + c), the group's
// products go through mma.sync into fp32, and the group's scale multiplies the fp32 sums. So nothing
// is rounded before the result. The inputs' order inside a block of 32 is the same permutation on both
// sides, which is why no shuffle is needed.
#pragma once
#include <cuda_fp16.h>

#include "api.h"
#include "common.cuh"

namespace msgl {

struct W4Tensor {
  const uint4* q;
  const uint32_t* s;  // two 16-bit scales
  const uint16_t* z;  // two zero points, or null
  int tiles, kb, kg, group, n, k, fp16;
};

inline W4Tensor w4_tensor(const MsglW4* w) {
  return {(const uint4*)w->q, (const uint32_t*)w->s, (const uint16_t*)w->z, w->tiles, w->kb, w->kg, w->group,
          w->n, w->k, w->fp16};
}

constexpr int kW4Warps = 16;
constexpr int kW4Threads = kW4Warps * 32;
constexpr int kW4Depth = 8;  // tiles of 512 bytes that a warp has in flight: 64 KB per SM

// a chunk is the least number of whole tiles and whole groups along the inputs
template <int G>
struct W4Chunk {
  static constexpr int kUnits = G == 128 ? 2 : 1;
  static constexpr int kScales = G == 32 ? 2 : 1;
  static constexpr int kDepth = kW4Depth / kUnits;
};

// shared memory of run_tiles for the warps' partial tiles
template <int NT>
constexpr int w4_part_bytes() { return kW4Warps * 2 * NT * 32 * 16; }

// bytes between the rows of the activations in shared memory: 64 more than a whole number of 128, so
// that the eight 16-byte reads of a quarter warp (two rows, four columns) fall into different banks
__host__ __device__ inline int w4_pitch(int inputs) { return inputs * 2 + 64; }

MSGL_DEVICE uint4 ld_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// asks for `bytes` (a multiple of 16, from a 16-byte boundary) to be brought into L2
MSGL_DEVICE void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

MSGL_DEVICE void mma_bf16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// two codes (bits 0-3 and 16-19 of v) minus a zero point (given as 128 + zero in both halves), exactly
MSGL_DEVICE uint32_t codes_bf16x2(uint32_t v, uint32_t zero) {
  uint32_t c;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(c) : "r"(v));  // (v & 0x000f000f) | 0x43004300
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&c), *reinterpret_cast<__nv_bfloat162*>(&zero));
  return *reinterpret_cast<const uint32_t*>(&d);
}

MSGL_DEVICE float2 w4_scales(uint32_t v, int fp16) {
  if (fp16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  return make_float2(bf16_lo(v), bf16_hi(v));
}

// A warp's run of chunks, fetched ahead in registers. Chunks are numbered tile by tile.
template <int G, bool Z>
struct W4Stream {
  using C = W4Chunk<G>;
  uint4 q[C::kDepth][C::kUnits];
  uint32_t s[C::kDepth][C::kScales];
  uint32_t z[Z ? C::kDepth : 1][C::kScales];
  const uint4* qp;
  const uint32_t* sp;
  const uint16_t* zp;
  int c, nc;            // next chunk of its tile, chunks per tile
  int q_skip, s_skip;   // from the end of a tile's chunks to the next tile's first

  MSGL_DEVICE void start(const W4Tensor& w, int64_t tile, int c0, int c_, int nc_) {
    const int lane = threadIdx.x & 31;
    const int64_t chunk = c0 + c_;
    c = c_;
    nc = nc_;
    qp = w.q + (tile * w.kb + chunk * C::kUnits) * 32 + lane;
    sp = w.s + (tile * w.kg + chunk * C::kScales) * 8 + (lane >> 2);
    zp = Z ? w.z + (tile * w.kg + chunk * C::kScales) * 8 + (lane >> 2) : nullptr;
    q_skip = (w.kb - nc * C::kUnits) * 32;
    s_skip = (w.kg - nc * C::kScales) * 8;
  }
  MSGL_DEVICE void fetch(int d) {
#pragma unroll
    for (int i = 0; i < C::kUnits; ++i) q[d][i] = ld_stream(qp + i * 32);
#pragma unroll
    for (int i = 0; i < C::kScales; ++i) {
      s[d][i] = __ldg(sp + i * 8);
      if constexpr (Z) z[d][i] = __ldg(zp + i * 8);
    }
    qp += C::kUnits * 32;
    sp += C::kScales * 8;
    if constexpr (Z) zp += C::kScales * 8;
    if (++c == nc) {
      c = 0;
      qp += q_skip;
      sp += s_skip;
      if constexpr (Z) zp += s_skip;
    }
  }
};

// Products of `ntiles` tiles (absolute number tile0 on) over chunks [c0, c0 + nc) with the nx rows in
// xs (pitch bytes apart, column 0 = chunk c0's first input). load() brings the rows into xs once the
// first weights are on their way; emit(tile, acc) gets every tile's sums, from one warp: acc[nt][0..3] =
// rows g, g, g + 8, g + 8 of tokens 8 nt + 2 t, + 1, + 0, + 1. Tiles that several warps share are summed
// through `part`, in the order of the warps. Ends without a barrier: xs is free, part is not until the
// next barrier.
template <int NT, int G, bool Z, class Load, class Emit>
MSGL_DEVICE void run_tiles(const W4Tensor& w, int64_t tile0, int ntiles, int c0, int nc, const uint8_t* xs, int pitch,
                           int nx, float4* part, Load load, Emit emit) {
  using C = W4Chunk<G>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t total = (int64_t)ntiles * nc;
  const auto bound = [&](int i) { return (int)(total * i / kW4Warps); };
  const int a = bound(warp), b = bound(warp + 1);
  int tile = a / nc, cc = a - tile * nc;
  const int tile_first = tile;
  W4Stream<G, Z> ws;
  ws.start(w, tile0 + tile, c0, cc, nc);
#pragma unroll
  for (int d = 0; d < C::kDepth; ++d)
    if (a + d < b) ws.fetch(d);
  load();
  __syncthreads();

  const uint8_t* xrow[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) xrow[nt] = xs + (size_t)min(nt * 8 + g, nx - 1) * pitch + t * 16;
  float acc[NT][4] = {};
  bool whole = cc == 0;  // the warp's part of this tile began at the tile's first chunk
  for (int i = a; i < b;) {
#pragma unroll
    for (int d = 0; d < C::kDepth; ++d) {
      if (i >= b) break;
      uint4 q[C::kUnits];
      uint32_t s[C::kScales], z[C::kScales];
#pragma unroll
      for (int u = 0; u < C::kUnits; ++u) q[u] = ws.q[d][u];
#pragma unroll
      for (int u = 0; u < C::kScales; ++u) {
        s[u] = ws.s[d][u];
        z[u] = Z ? ws.z[d][u] : 0x0808u;
      }
      if (i + C::kDepth < b) ws.fetch(d);
      float tmp[NT][4];
#pragma unroll
      for (int u = 0; u < C::kUnits; ++u) {
        const uint32_t words[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int si = C::kScales == 2 ? h : 0;
          const uint32_t z0 = Z ? 0x43004300u + (z[si] & 15u) * 0x10001u : 0x43084308u;
          const uint32_t z1 = Z ? 0x43004300u + ((z[si] >> 8) & 15u) * 0x10001u : 0x43084308u;
          if (G == 32 || (h == 0 && u == 0)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int r = 0; r < 4; ++r) tmp[nt][r] = 0.f;
          }
          uint32_t fr[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t v = words[2 * h + j];
            fr[j][0] = codes_bf16x2(v, z0);
            fr[j][1] = codes_bf16x2(v >> 4, z1);
            fr[j][2] = codes_bf16x2(v >> 8, z0);
            fr[j][3] = codes_bf16x2(v >> 12, z1);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 xv = *reinterpret_cast<const uint4*>(xrow[nt] + (cc * C::kUnits + u) * 128 + h * 64);
            mma_bf16_16816(tmp[nt], fr[0], xv.x, xv.y);
            mma_bf16_16816(tmp[nt], fr[1], xv.z, xv.w);
          }
          if (G == 32 || (h == 1 && u == C::kUnits - 1)) {
            const float2 sc = w4_scales(s[si], w.fp16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              acc[nt][0] += tmp[nt][0] * sc.x;
              acc[nt][1] += tmp[nt][1] * sc.x;
              acc[nt][2] += tmp[nt][2] * sc.y;
              acc[nt][3] += tmp[nt][3] * sc.y;
            }
          }
        }
      }
      ++i;
      ++cc;
      if (cc == nc || i == b) {
        if (cc == nc && whole) {
          emit(tile, acc);
        } else {
          float4* p = part + ((warp * 2 + (tile == tile_first ? 0 : 1)) * NT) * 32 + lane;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) p[nt * 32] = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[nt][r] = 0.f;
        whole = true;
        if (cc == nc) {
          cc = 0;
          ++tile;
        }
      }
    }
  }
  __syncthreads();
  // a tile that starts in this warp's run and ends in a later warp's: sum their parts in order
  if (a < b) {
    const int last = (b - 1) / nc;
    const int64_t from = (int64_t)last * nc, to = from + nc;
    if (a <= from && b < to) {
      const float4* p = part + ((warp * 2 + (last == tile_first ? 0 : 1)) * NT) * 32 + lane;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float4 v = p[nt * 32];
        acc[nt][0] = v.x, acc[nt][1] = v.y, acc[nt][2] = v.z, acc[nt][3] = v.w;
      }
      for (int v = warp + 1; v < kW4Warps && bound(v) < to; ++v) {
        if (bound(v) == bound(v + 1)) continue;
        const float4* o = part + (v * 2 * NT) * 32 + lane;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float4 f = o[nt * 32];
          acc[nt][0] += f.x, acc[nt][1] += f.y, acc[nt][2] += f.z, acc[nt][3] += f.w;
        }
      }
      emit(last, acc);
    }
  }
}

// rows of bf16 activations into shared memory: row(r) gives row r's address; inputs [k0, k0 + kn) of k,
// zeros beyond k
template <class Row>
MSGL_DEVICE void load_rows(uint8_t* xs, int pitch, int nx, int k0, int kn, int k, Row row) {
  const int vec = kn / 8;
  for (int r = threadIdx.x >> 5; r < nx; r += kW4Warps) {
    const __nv_bfloat16* src = row(r) + k0;
    for (int i = threadIdx.x & 31; i < vec; i += 32) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (k0 + i * 8 < k) v = *reinterpret_cast<const uint4*>(src + i * 8);
      *reinterpret_cast<uint4*>(xs + (size_t)r * pitch + i * 16) = v;
    }
  }
}

}  // namespace msgl
