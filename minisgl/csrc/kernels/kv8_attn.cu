// Ragged causal attention over the paged 8-bit cache:
//
//   o_i = sum_j w_ij s^v_j c^v_j / sum_j w_ij,  w_ij = exp(scale s^k_j q_i . c^k_j),  over the keys j that query i sees
#include "kv8_stream.cuh"
#include "kv8_tiles.cuh"

#include <mutex>

using namespace msgl;

namespace {

typedef CUresult (*Kv8EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Kv8EncodeFn encode_fn() {
  static Kv8EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<Kv8EncodeFn>(ptr);
  });
  return fn;
}

// Keys' and values' tensors as one, its last dimension the way from the one to the other, in boxes of a page of one head
// of both: codes [2][nkv][slots][HD], rows of HD bytes swizzled, and scales [2][nkv][slots].
bool encode_cache(CUtensorMap* tc, CUtensorMap* ts, Kv8Order* order, const Kv8Attn& p, int hd) {
  const Kv8EncodeFn fn = encode_fn();
  const char *k = (const char*)p.ck, *v = (const char*)p.cv, *sk = (const char*)p.sk, *sv = (const char*)p.sv;
  if (fn == nullptr) return false;
  order->codes = k < v ? 0 : 1;
  order->scales = sk < sv ? 0 : 1;
  const cuuint32_t ones[4] = {1, 1, 1, 1}, page = (cuuint32_t)p.page;
  const cuuint64_t slots = (cuuint64_t)p.num_slots, heads = (cuuint64_t)p.nkv;
  const cuuint64_t cdims[4] = {(cuuint64_t)hd, slots, heads, 2}, sdims[3] = {slots, heads, 2};
  const cuuint64_t cstr[3] = {(cuuint64_t)hd, hd * slots, (cuuint64_t)(k < v ? v - k : k - v)};
  const cuuint64_t sstr[2] = {4 * slots, (cuuint64_t)(sk < sv ? sv - sk : sk - sv)};
  const cuuint32_t cbox[4] = {(cuuint32_t)hd, page, 1, 2}, sbox[3] = {page, 1, 2};
  return fn(tc, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<char*>(k < v ? k : v), cdims, cstr, cbox, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS &&
         fn(ts, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<char*>(sk < sv ? sk : sv), sdims, sstr, sbox, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Queries [total_q][nq][HD] bf16 in boxes of 64 head dims of the heads of a group, of as many tokens as a tile holds.
bool encode_queries(CUtensorMap* m, const Kv8Attn& p, int hd) {
  const Kv8EncodeFn fn = encode_fn();
  if (fn == nullptr) return false;
  const int G = p.nq / p.nkv;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)p.nq, (cuuint64_t)p.total_q};
  const cuuint64_t strides[2] = {(cuuint64_t)p.q_head * 2, (cuuint64_t)p.q_row * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(128 / G)}, ones[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <int HD, bool FP8, int NR>
int stream_form(const Kv8Attn& p, void* ws, int* launches, cudaStream_t s) {
  using C = KsCfg<HD, NR>;
  constexpr auto kernel = kv8_stream_kernel<HD, FP8, NR>;
  if (msgl_set_smem<kernel>(C::kSmem, 100) != cudaSuccess) return 4;
  CUtensorMap tc, ts;
  Kv8Order order;
  if (!encode_cache(&tc, &ts, &order, p, HD)) return 2;
  const int ctas = 2 * sm_count();
  const Kv8Scratch scratch = kv8_scratch<C::kRows, HD>(ws, ctas);
  if (msgl_launch(kernel, dim3(ctas), dim3(kKsThreads), C::kSmem, s, 1, tc, ts, p, order, scratch) != cudaSuccess) return 4;
  ++*launches;
  if (msgl_launch(kv8_join_kernel<C::kRows, HD>, dim3(ctas, C::kRows / 4), dim3(128), 0, s, 1, p, scratch) != cudaSuccess) return 4;
  ++*launches;
  return 0;
}

template <int HD, bool FP8>
int tiles_form(const Kv8Attn& p, void* ws, int* launches, cudaStream_t s) {
  using C = KtCfg<HD>;
  constexpr auto kernel = kv8_tiles_kernel<HD, FP8>;
  if (msgl_set_smem<kernel>(C::kSmem) != cudaSuccess) return 4;
  // (the roles' registers have to fit the launch's, or a warp would wait for more of them for good)
  static const bool fits = [] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kernel) == cudaSuccess && a.numRegs >= kKtRegs;
  }();
  if (!fits) return 4;
  CUtensorMap tc, ts, tq;
  Kv8Order order;
  if (!encode_cache(&tc, &ts, &order, p, HD) || !encode_queries(&tq, p, HD)) return 2;
  const int ctas = sm_count();
  const Kv8Scratch scratch = kv8_scratch<kKtRows, HD>(ws, ctas);
  if (msgl_launch(kernel, dim3(ctas), dim3(kKtThreads), C::kSmem, s, 1, tc, ts, tq, p, order, scratch) != cudaSuccess) return 4;
  ++*launches;
  // (32: two rows a warp; 8 take 7 us longer after short prompts, 64 start too many blocks where few are cut)
  if (msgl_launch(kv8_join_kernel<kKtRows, HD>, dim3(ctas, 32), dim3(128), 0, s, 1, p, scratch) != cudaSuccess) return 4;
  ++*launches;
  return 0;
}

// The form for what the caller has told of a request's rows: 8, 16: rows of a streaming tile, 256: tensor core tiles. A request
// of more rows than a streaming tile has its keys streamed (out of the L2 cache) and converted once for each tile,
// which the tensor core form does once for 256 rows, but at its own pace. Measured with 16 requests of 6000 keys, 8 kv heads, int8, us
// by rows, tiles of 8, of 16, tensor core: head dim 128: 8: 47, 58, 114; 16: 78, 59, 114; 32: 143, 101, 116; 48: 208, 144, 122;
// 64: 273, 187, 125; head dim 64: 8: 35, 41, 110; 16: 58, 42, 109; 48: 151, 99, 115; 64: 197, 128, 114. (A single request of
// 4000 keys takes 13 to 27 us in tiles of 16 up to 128 rows, 30 to 42 on the tensor core from 64 rows on.)
int form_of(const Kv8Attn& p, int hd, int max_q_len) {
  const int64_t rows = (int64_t)max_q_len * (p.nq / p.nkv);
  return rows <= 8 ? 8 : rows <= (hd == 128 ? 32 : 48) ? 16 : 256;
}

template <int HD, bool FP8>
int any_form(const Kv8Attn& p, int max_q_len, void* ws, int* launches, cudaStream_t s) {
  switch (form_of(p, HD, max_q_len)) {
    case 8: return stream_form<HD, FP8, 1>(p, ws, launches, s);
    case 16: return stream_form<HD, FP8, 2>(p, ws, launches, s);
    default: return tiles_form<HD, FP8>(p, ws, launches, s);
  }
}

template <int HD>
int64_t workspace(int form) {
  const int sms = sm_count();
  return form == 8 ? kv8_scratch_bytes<8, HD>(2 * sms) : form == 16 ? kv8_scratch_bytes<16, HD>(2 * sms) : kv8_scratch_bytes<kKtRows, HD>(sms);
}

}  // namespace

extern "C" int64_t msgl_kv8_attention_workspace(const Kv8Attn* p, int hd, int max_q_len) {
  return hd == 128 ? workspace<128>(form_of(*p, hd, max_q_len)) : workspace<64>(form_of(*p, hd, max_q_len));
}

extern "C" int msgl_kv8_attention(const Kv8Attn* args, int hd, int fp8, int max_q_len, void* ws, int* launches, cudaStream_t s) {
  *launches = 0;
  Kv8Attn p = *args;
  // with s = 30 + ceil(log2 G) and mul = ceil(2^s / G), x mul / 2^s is x / G and less than x / 2^s more, too little to reach
  // the next whole number
  const uint64_t G = p.nq / p.nkv;
  p.group_shift = 30;
  while ((G << 30) > (1ull << p.group_shift)) ++p.group_shift;
  p.group_mul = (unsigned)(((1ull << p.group_shift) + G - 1) / G);
  if (hd == 128) return fp8 ? any_form<128, true>(p, max_q_len, ws, launches, s) : any_form<128, false>(p, max_q_len, ws, launches, s);
  if (hd == 64) return fp8 ? any_form<64, true>(p, max_q_len, ws, launches, s) : any_form<64, false>(p, max_q_len, ws, launches, s);
  return 3;
}

MSGL_ERROR_ACCESSOR(msgl_err_kv8_attn)
