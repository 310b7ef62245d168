// 8-bit key/value cache: quantising rows as they are written, and reading them back.
//
// Layout (per layer): codes [kv heads][slots][HD] bytes and fp32 scales [kv heads][slots], of keys and of
// values: a head's page is one contiguous run of codes and one of scales, so attention loads it with one
// copy each.
#include "api.h"
#include "common.cuh"
#include "kv8.cuh"

using namespace msgl;

namespace {

constexpr int kThreads = 256;

// x / nkv for x < 2^31 (head_mul and head_shift by divide_by)
MSGL_DEVICE int by_heads(uint32_t x, uint32_t mul, uint32_t shift) { return (int)((uint64_t)x * mul >> shift); }

// A block takes the rows of one head of kThreads / (HD / 8) tokens, HD / 8 lanes per row, 8 values each of the key's and of the
// value's: 16-byte loads of whole rows, 8-byte stores of whole 128- (64-) byte code rows, next to one another where slots are.
// Both rows' largest magnitudes go through the lanes at once. Bound by instructions as much as by memory: 16384
// tokens of 8 heads of 128 take 20 us, 5.1 TB/s (28.8 us with a division per value's row, __fdiv_rn and one value at a time in
// the quotients; 21.4 us with the rows of a token's heads in a block). One token: 1.6 us in a graph.
template <int HD, bool FP8>
__global__ void __launch_bounds__(kThreads) kv8_store_kernel(Kv8Store p, uint32_t head_mul, uint32_t head_shift) {
  pdl_wait();
  pdl_launch();
  constexpr int L = HD / 8;
  const int group = by_heads(blockIdx.x, head_mul, head_shift), h = (int)blockIdx.x - group * p.nkv;
  const int64_t token = (int64_t)group * (kThreads / L) + threadIdx.x / L;
  const int part = threadIdx.x % L;
  const bool in = token < p.n;
  const int64_t t = in ? token : 0;
  uint4 u[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(i ? p.v : p.k) +
                               (i ? t * p.v_row + h * p.v_head : t * p.k_row + h * p.k_head);
    u[i] = in ? __ldcs(reinterpret_cast<const uint4*>(src) + part) : make_uint4(0, 0, 0, 0);
  }
  int slot = in ? p.slots[t] : -1;
  if (slot >= p.num_slots) {
    report_error(kErrBounds, kBcKvSlot);
    slot = -1;
  }
  // the largest magnitudes, the key's in the low half: with the sign gone bf16 patterns order as integers, infinities and NaN on top
  uint32_t top[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    top[i] = __vmaxu2(__vmaxu2(u[i].x & 0x7fff7fffu, u[i].y & 0x7fff7fffu), __vmaxu2(u[i].z & 0x7fff7fffu, u[i].w & 0x7fff7fffu));
  uint32_t m = __vmaxu2(__byte_perm(top[0], top[1], 0x5410), __byte_perm(top[0], top[1], 0x7632));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (slot < 0) return;
  const int64_t at = (int64_t)h * p.num_slots + slot;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const Kv8Quant<FP8> quant(i ? bf16_hi(m) : bf16_lo(m));
    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = quant.pair(bf16_lo(w[j]), bf16_hi(w[j]));
    reinterpret_cast<uint2*>(i ? p.cv : p.ck)[at * L + part] =
        make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
    if (part == 0) (i ? p.sv : p.sk)[at] = quant.scale;
  }
}

// HD / 8 lanes per row, keys and values at once, U rows per lane, all loaded before the first is stored. Bound by DRAM: 120000 tokens
// of 8 heads of 128 take 116 us, 6.4 TB/s, with U = 2 (127 us with 1, 117 with 3; 11 us more without the streaming hints).
// Few rows (below 16 blocks of U = 1 per SM) spread better with U = 1.
template <int HD, bool FP8, int U>
__global__ void __launch_bounds__(kThreads) kv8_load_kernel(Kv8Load p, uint32_t head_mul, uint32_t head_shift) {
  pdl_wait();
  pdl_launch();
  constexpr int L = HD / 8;
  const uint32_t row0 = blockIdx.x * (kThreads * U / L) + threadIdx.x / L, rows = (uint32_t)p.n * p.nkv;
  const int part = threadIdx.x % L;
  uint2 c[U][2];
  float s[U][2];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const uint32_t row = row0 + j * (kThreads / L);
    const bool in = row < rows;
    const int t = in ? by_heads(row, head_mul, head_shift) : 0, h = in ? (int)row - t * p.nkv : 0;
    int slot = in ? p.slots[t] : -1;
    if (slot >= p.num_slots) {
      report_error(kErrBounds, kBcKvSlot);
      slot = -1;
    }
    c[j][0] = c[j][1] = make_uint2(0, 0);
    s[j][0] = s[j][1] = 0.f;
    if (slot >= 0) {
      const int64_t at = (int64_t)h * p.num_slots + slot;
      c[j][0] = __ldcs(reinterpret_cast<const uint2*>(p.ck) + at * L + part);
      c[j][1] = __ldcs(reinterpret_cast<const uint2*>(p.cv) + at * L + part);
      s[j][0] = __ldg(p.sk + at);
      s[j][1] = __ldg(p.sv + at);
    }
  }
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const uint32_t row = row0 + j * (kThreads / L);
    if (row >= rows) break;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 f = kv8_decode2<FP8>((q & 2 ? c[j][i].y : c[j][i].x) >> (16 * (q & 1)));
        w[q] = pack_bf16(f.x * s[j][i], f.y * s[j][i]);
      }
      __stcs(reinterpret_cast<uint4*>(i ? p.v : p.k) + (int64_t)row * L + part, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
}

// x / by = x mul >> shift for x < 2^31 and by < 2^31: with shift = 31 + ceil(log2 by) and mul = ceil(2^shift / by) the product is x / by and less
// than x / 2^shift more, too little to reach the next whole number
void divide_by(uint64_t by, uint32_t* mul, uint32_t* shift) {
  *shift = 31;
  while ((by << 31) > (1ull << *shift)) ++*shift;
  *mul = (uint32_t)(((1ull << *shift) + by - 1) / by);
}

}  // namespace

extern "C" int msgl_kv8_store(const Kv8Store* p, int hd, int fp8, cudaStream_t s) {
  const int64_t per = kThreads / (hd / 8), blocks = ((int64_t)p->n + per - 1) / per * p->nkv;
  if ((hd != 64 && hd != 128) || blocks > INT32_MAX) return 3;
  if (blocks == 0) return 0;
  uint32_t mul, shift;
  divide_by(p->nkv, &mul, &shift);
  auto* f = hd == 64 ? (fp8 ? kv8_store_kernel<64, true> : kv8_store_kernel<64, false>)
                     : (fp8 ? kv8_store_kernel<128, true> : kv8_store_kernel<128, false>);
  return msgl_launch(f, dim3((unsigned)blocks), dim3(kThreads), 0, s, 1, *p, mul, shift) == cudaSuccess ? 0 : 4;
}

template <int U>
static int load_rows(const Kv8Load* p, int hd, int fp8, cudaStream_t s) {
  const int64_t rows = (int64_t)p->n * p->nkv, per = kThreads * U / (hd / 8);
  uint32_t mul, shift;
  divide_by(p->nkv, &mul, &shift);
  auto* f = hd == 64 ? (fp8 ? kv8_load_kernel<64, true, U> : kv8_load_kernel<64, false, U>)
                     : (fp8 ? kv8_load_kernel<128, true, U> : kv8_load_kernel<128, false, U>);
  return msgl_launch(f, dim3((unsigned)((rows + per - 1) / per)), dim3(kThreads), 0, s, 1, *p, mul, shift) == cudaSuccess ? 0 : 4;
}

extern "C" int msgl_kv8_load(const Kv8Load* p, int hd, int fp8, cudaStream_t s) {
  const int64_t rows = (int64_t)p->n * p->nkv;
  if ((hd != 64 && hd != 128) || rows > INT32_MAX - 2 * kThreads) return 3;
  if (rows == 0) return 0;
  return rows * (hd / 8) < 148 * 16 * kThreads ? load_rows<1>(p, hd, fp8, s) : load_rows<2>(p, hd, fp8, s);
}

MSGL_ERROR_ACCESSOR(msgl_err_kv8)
