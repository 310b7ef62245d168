// Ragged causal attention over the paged 8-bit cache:
//
//   o_i = sum_j w_ij s^v_j c^v_j / sum_j w_ij,  w_ij = exp(scale s^k_j q_i . c^k_j),  over the keys j that query i sees
#include "kv8_stream.cuh"

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

int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <int HD, bool FP8>
int stream_form(const Kv8Attn& p, void* ws, int* launches, cudaStream_t s) {
  using C = KsCfg<HD>;
  constexpr auto kernel = kv8_stream_kernel<HD, FP8>;
  if (msgl_set_smem<kernel>(C::kSmem, 100) != cudaSuccess) return 4;
  CUtensorMap tc, ts;
  Kv8Order order;
  if (!encode_cache(&tc, &ts, &order, p, HD)) return 2;
  const int ctas = 2 * sm_count();
  const Kv8Scratch scratch = kv8_scratch<kKsRows, HD>(ws, ctas);
  if (msgl_launch(kernel, dim3(ctas), dim3(kKsThreads), C::kSmem, s, 1, tc, ts, p, order, scratch) != cudaSuccess) return 4;
  ++*launches;
  if (msgl_launch(kv8_join_kernel<kKsRows, HD>, dim3(ctas, kKsRows / 4), dim3(128), 0, s, 1, p, scratch) != cudaSuccess) return 4;
  ++*launches;
  return 0;
}

}  // namespace

extern "C" int64_t msgl_kv8_attention_workspace(const Kv8Attn* p, int hd, int max_q_len) {
  (void)p, (void)max_q_len;
  const int ctas = 2 * sm_count();
  return hd == 128 ? kv8_scratch_bytes<kKsRows, 128>(ctas) : kv8_scratch_bytes<kKsRows, 64>(ctas);
}

extern "C" int msgl_kv8_attention(const Kv8Attn* p, int hd, int fp8, int max_q_len, void* ws, int* launches, cudaStream_t s) {
  (void)max_q_len;
  *launches = 0;
  if (hd == 128) return fp8 ? stream_form<128, true>(*p, ws, launches, s) : stream_form<128, false>(*p, ws, launches, s);
  if (hd == 64) return fp8 ? stream_form<64, true>(*p, ws, launches, s) : stream_form<64, false>(*p, ws, launches, s);
  return 3;
}

MSGL_ERROR_ACCESSOR(msgl_err_kv8_attn)
