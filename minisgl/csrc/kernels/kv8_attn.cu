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

// Codes [nkv][slots][HD] in boxes of a page of one head, rows of HD bytes swizzled.
bool encode_codes(CUtensorMap* m, const void* codes, const Kv8Attn& p, int hd) {
  static Kv8EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<Kv8EncodeFn>(ptr);
  });
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)p.num_slots, (cuuint64_t)p.nkv};
  const cuuint64_t strides[2] = {(cuuint64_t)hd, (cuuint64_t)hd * p.num_slots};
  const cuuint32_t box[3] = {(cuuint32_t)hd, (cuuint32_t)p.page, 1}, ones[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
  if (msgl_set_smem<kernel>(C::kSmem) != cudaSuccess) return 4;
  CUtensorMap tk, tv;
  if (!encode_codes(&tk, p.ck, p, HD) || !encode_codes(&tv, p.cv, p, HD)) return 2;
  const int ctas = sm_count();
  const Kv8Scratch scratch = kv8_scratch<kKsRows, HD>(ws, ctas);
  if (msgl_launch(kernel, dim3(ctas), dim3(kKsThreads), C::kSmem, s, 1, tk, tv, p, scratch) != cudaSuccess) return 4;
  ++*launches;
  if (msgl_launch(kv8_join_kernel<kKsRows, HD>, dim3(ctas, kKsRows / 8), dim3(256), 0, s, 1, p, scratch) != cudaSuccess) return 4;
  ++*launches;
  return 0;
}

}  // namespace

extern "C" int64_t msgl_kv8_attention_workspace(const Kv8Attn* p, int hd, int max_q_len) {
  (void)p, (void)max_q_len;
  return hd == 128 ? kv8_scratch_bytes<kKsRows, 128>(sm_count()) : kv8_scratch_bytes<kKsRows, 64>(sm_count());
}

extern "C" int msgl_kv8_attention(const Kv8Attn* p, int hd, int fp8, int max_q_len, void* ws, int* launches, cudaStream_t s) {
  (void)max_q_len;
  *launches = 0;
  if (hd == 128) return fp8 ? stream_form<128, true>(*p, ws, launches, s) : stream_form<128, false>(*p, ws, launches, s);
  if (hd == 64) return fp8 ? stream_form<64, true>(*p, ws, launches, s) : stream_form<64, false>(*p, ws, launches, s);
  return 3;
}

MSGL_ERROR_ACCESSOR(msgl_err_kv8_attn)
