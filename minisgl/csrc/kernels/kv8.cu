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

// HD / 8 lanes per row of a token and a head, 8 values each, the key's and the value's row one after the other:
// 16-byte loads of whole rows, 8-byte stores of whole 128- (64-) byte code rows. Bound by DRAM.
template <int HD, bool FP8>
__global__ void __launch_bounds__(kThreads) kv8_store_kernel(Kv8Store p) {
  pdl_wait();
  pdl_launch();
  constexpr int L = HD / 8;
  const int64_t row = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  const int part = threadIdx.x % L;
  const bool in = row < (int64_t)p.n * p.nkv;
  const int t = in ? (int)(row / p.nkv) : 0, h = in ? (int)(row - (int64_t)t * p.nkv) : 0;
  int slot = in ? p.slots[t] : -1;
  if (slot >= p.num_slots) {
    report_error(kErrBounds, kBcKvSlot);
    slot = -1;
  }
  uint4 u[2];
  float top[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(i ? p.v : p.k) +
                               (i ? t * p.v_row + h * p.v_head : t * p.k_row + h * p.k_head);
    u[i] = in ? __ldg(reinterpret_cast<const uint4*>(src) + part) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // the largest magnitude: with the sign gone bf16 patterns order as integers, infinities and NaN on top
    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = max(m & 0xffffu, m >> 16);
    top[i] = __uint_as_float(m << 16);
  }
  if (slot < 0) return;
  const int64_t at = (int64_t)h * p.num_slots + slot;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const Kv8Quant<FP8> quant(top[i]);
    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = quant.pair(bf16_lo(w[j]), bf16_hi(w[j]));
    reinterpret_cast<uint2*>(i ? p.cv : p.ck)[at * L + part] = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    if (part == 0) (i ? p.sv : p.sk)[at] = quant.scale;
  }
}

// One row per HD / 8 lanes, keys and values at once. Bound by DRAM.
template <int HD, bool FP8>
__global__ void __launch_bounds__(kThreads) kv8_load_kernel(Kv8Load p) {
  pdl_wait();
  pdl_launch();
  constexpr int L = HD / 8;
  const int64_t row = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  const int part = threadIdx.x % L;
  if (row >= (int64_t)p.n * p.nkv) return;
  const int t = (int)(row / p.nkv), h = (int)(row - (int64_t)t * p.nkv);
  int slot = p.slots[t];
  if (slot >= p.num_slots) {
    report_error(kErrBounds, kBcKvSlot);
    slot = -1;
  }
  uint2 c[2] = {make_uint2(0, 0), make_uint2(0, 0)};
  float s[2] = {0.f, 0.f};
  if (slot >= 0) {
    const int64_t at = (int64_t)h * p.num_slots + slot;
    c[0] = __ldg(reinterpret_cast<const uint2*>(p.ck) + at * L + part);
    c[1] = __ldg(reinterpret_cast<const uint2*>(p.cv) + at * L + part);
    s[0] = __ldg(p.sk + at);
    s[1] = __ldg(p.sv + at);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = kv8_decode2<FP8>((j & 2 ? c[i].y : c[i].x) >> (16 * (j & 1)));
      w[j] = pack_bf16(f.x * s[i], f.y * s[i]);
    }
    reinterpret_cast<uint4*>(i ? p.v : p.k)[row * L + part] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace

extern "C" int msgl_kv8_store(const Kv8Store* p, int hd, int fp8, cudaStream_t s) {
  const int64_t blocks = ((int64_t)p->n * p->nkv * (hd / 8) + kThreads - 1) / kThreads;
  if ((hd != 64 && hd != 128) || blocks > INT32_MAX) return 3;
  if (blocks == 0) return 0;
  auto* f = hd == 64 ? (fp8 ? kv8_store_kernel<64, true> : kv8_store_kernel<64, false>)
                     : (fp8 ? kv8_store_kernel<128, true> : kv8_store_kernel<128, false>);
  return msgl_launch(f, dim3((unsigned)blocks), dim3(kThreads), 0, s, 1, *p) == cudaSuccess ? 0 : 4;
}

extern "C" int msgl_kv8_load(const Kv8Load* p, int hd, int fp8, cudaStream_t s) {
  const int64_t blocks = ((int64_t)p->n * p->nkv * (hd / 8) + kThreads - 1) / kThreads;
  if ((hd != 64 && hd != 128) || blocks > INT32_MAX) return 3;
  if (blocks == 0) return 0;
  auto* f = hd == 64 ? (fp8 ? kv8_load_kernel<64, true> : kv8_load_kernel<64, false>)
                     : (fp8 ? kv8_load_kernel<128, true> : kv8_load_kernel<128, false>);
  return msgl_launch(f, dim3((unsigned)blocks), dim3(kThreads), 0, s, 1, *p) == cudaSuccess ? 0 : 4;
}

MSGL_ERROR_ACCESSOR(msgl_err_kv8)
