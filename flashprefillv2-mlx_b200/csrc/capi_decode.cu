// C ABI of the decode step (declared in include/fpv2_b200.h): argument checks
// and launches, as in capi.cu.
#include <cmath>
#include <string>

#include "../../include/fpv2_b200.h"
#include "common.cuh"
#include "kernels.h"

namespace fpv2 {
namespace {

int invalid(const char* msg) { return report_error(FPV2_ERR_INVALID_ARGUMENT, msg); }

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return FPV2_OK;
  return report_error(FPV2_ERR_CUDA, (std::string(what) + ": " + cudaGetErrorString(e)).c_str());
}

bool half_type(int dt) { return dt == DT_F16 || dt == DT_BF16; }

bool multiple(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace fpv2

using namespace fpv2;

extern "C" {

int fpv2_qk_norm_rope(const void* q, const void* k, const void* v, int dtype, int64_t tokens,
                      int32_t q_heads, int32_t kv_heads, int32_t head_dim, const int64_t* in_strides,
                      const void* positions, int32_t positions_int64, const float* table,
                      int64_t table_positions, int32_t rotary_dim, int32_t interleaved,
                      const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                      void* q_out, void* k_out, const int64_t* out_strides, void* k_cache,
                      void* v_cache, const int64_t* cache_strides, const int64_t* slots,
                      int64_t num_pages, int32_t page_size, void* stream) {
  if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32) return invalid("unknown dtype code");
  if ((q_weight || k_weight) && weight_dtype != DT_F16 && weight_dtype != DT_BF16 && weight_dtype != DT_F32)
    return invalid("unknown weight dtype code");
  if (tokens < 0 || q_heads <= 0 || kv_heads <= 0) return invalid("invalid shape");
  if (head_dim <= 0 || head_dim > 256) return invalid("head dimension must be in [1, 256]");
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return invalid("rotary_dim must be even and in [2, head_dim]");
  if (table_positions <= 0) return invalid("the rotation table is empty");
  if (!(eps >= 0.f) || std::isinf(eps)) return invalid("eps must be finite and non-negative");
  const bool paged = k_cache != nullptr || v_cache != nullptr;
  if (paged && (!k_cache || !v_cache || !slots || num_pages <= 0 || page_size <= 0))
    return invalid("a cache needs k and v pages, a page size and slots");
  if (!in_strides || !out_strides || (paged && !cache_strides)) return invalid("null stride array");
  if (tokens == 0) return FPV2_OK;
  if (!q || !k || !positions || !table || !q_out || (paged ? !v : !k_out)) return invalid("null tensor pointer");
  TcLaunch L;
  const int rc = current_launch(&L);
  if (rc != FPV2_OK) return rc;
  RopeArgs a = {};
  a.q = q;
  a.k = k;
  a.v = paged ? v : nullptr;
  a.q_st = in_strides[0];
  a.q_sh = in_strides[1];
  a.k_st = in_strides[2];
  a.k_sh = in_strides[3];
  a.v_st = paged ? in_strides[4] : 0;
  a.v_sh = paged ? in_strides[5] : 0;
  a.positions = positions;
  a.pos64 = positions_int64 ? 1 : 0;
  a.table = table;
  a.max_pos = table_positions;
  a.rot = rotary_dim;
  a.interleaved = interleaved ? 1 : 0;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.weight_dt = weight_dtype;
  a.eps = eps;
  a.q_out = q_out;
  a.qo_st = out_strides[0];
  a.qo_sh = out_strides[1];
  if (paged) {
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.kc_sp = cache_strides[0];
    a.kc_sr = cache_strides[1];
    a.kc_sh = cache_strides[2];
    a.vc_sp = cache_strides[3];
    a.vc_sr = cache_strides[4];
    a.vc_sh = cache_strides[5];
    a.slots = slots;
    a.page_size = page_size;
    a.num_slots = num_pages * page_size;
  } else {
    a.k_out = k_out;
    a.ko_st = out_strides[2];
    a.ko_sh = out_strides[3];
  }
  a.tokens = tokens;
  a.Hq = q_heads;
  a.Hkv = kv_heads;
  a.D = head_dim;
  return launched(launch_qk_rope(a, dtype, L.num_sms, reinterpret_cast<cudaStream_t>(stream)),
                  "qk_norm_rope launch");
}

int64_t fpv2_decode_workspace_bytes(int32_t new_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (new_tokens <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || !decode_supported(head_dim))
    return 0;
  return (int64_t)decode_workspace_bytes(new_tokens, q_heads, kv_heads, head_dim);
}

int fpv2_decode_attention(const void* q, const void* k_pages, const void* v_pages, int dtype,
                          int32_t batch, int32_t new_tokens, int32_t q_heads, int32_t kv_heads,
                          int32_t head_dim, const int64_t* strides, const int32_t* block_tables,
                          int64_t table_stride, int32_t table_width, const int32_t* lengths,
                          int32_t num_pages, int32_t page_size, float scale, int32_t window,
                          int32_t sinks, void* out, float* lse, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  if (!half_type(dtype)) return invalid("q and the caches must share float16 or bfloat16 dtype");
  if (batch < 0 || new_tokens <= 0) return invalid("invalid shape");
  if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads)
    return invalid("query heads must be divisible by KV heads");
  if ((int64_t)q_heads * new_tokens > (1 << 24)) return invalid("too many query rows a sequence");
  if (!decode_supported(head_dim)) return invalid("head dimension must be 64, 96, 128 or 256");
  if (num_pages <= 0 || page_size <= 0 || table_width <= 0)
    return invalid("paged K/V needs block tables, pages and a page size");
  if ((int64_t)table_width * page_size > 0x7fffffff - 64) return invalid("sequences must be shorter than 2^31 keys");
  if (window < 0 || sinks < 0) return invalid("window and sinks must be non-negative");
  if (!std::isfinite(scale)) return invalid("scale must be finite");
  if (!strides) return invalid("null stride array");
  if (batch == 0) return FPV2_OK;
  if (!q || !k_pages || !v_pages || !block_tables || !lengths || !out || !workspace)
    return invalid("null tensor pointer");
  if (!multiple(workspace, 16) ||
      workspace_bytes < (int64_t)decode_workspace_bytes(new_tokens, q_heads, kv_heads, head_dim))
    return invalid("workspace is too small or not 16-byte aligned");
  for (int i = 0; i < 9; ++i)
    if (strides[i] % (i < 3 ? 2 : 8)) return invalid("q strides must be multiples of 2 elements, cache strides of 8");
  if (!multiple(q, 4) || !multiple(out, 4) || !multiple(k_pages, 16) || !multiple(v_pages, 16))
    return invalid("q and out must be 4-byte aligned, the caches 16-byte");
  TcLaunch L;
  const int rc = current_launch(&L);
  if (rc != FPV2_OK) return rc;
  DecodeArgs a = {};
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.q_sb = strides[0];
  a.q_st = strides[1];
  a.q_sh = strides[2];
  a.k_sp = strides[3];
  a.k_sr = strides[4];
  a.k_sh = strides[5];
  a.v_sp = strides[6];
  a.v_sr = strides[7];
  a.v_sh = strides[8];
  a.tables = block_tables;
  a.lengths = lengths;
  a.table_stride = table_stride;
  a.B = batch;
  a.T = new_tokens;
  a.Hq = q_heads;
  a.Hkv = kv_heads;
  a.G = q_heads / kv_heads;
  a.D = head_dim;
  a.num_pages = num_pages;
  a.page_size = page_size;
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (page_size == 1 << i) a.page_shift = i;
  a.table_width = table_width;
  a.window = window;
  a.sinks = sinks;
  a.scale_log2 = scale * kLog2e;
  a.out = out;
  a.lse = lse;
  a.workspace = workspace;
  a.status = L.status;
  return launched(launch_decode(a, dtype, reinterpret_cast<cudaStream_t>(stream)), "decode_attention launch");
}

int fpv2_sample_tokens(const void* logits, int dtype, int64_t rows, int32_t vocab, int64_t logits_stride,
                       const float* noise, int64_t noise_stride, const float* temperature,
                       float temperature_all, const int32_t* top_k, int32_t top_k_all,
                       const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                       int64_t* tokens, float* logprobs, void* stream) {
  if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32) return invalid("unknown dtype code");
  if (rows < 0 || rows > (1 << 24) || vocab <= 0 || vocab > (1 << 30)) return invalid("invalid shape");
  if (rows == 0) return FPV2_OK;
  if (!logits || !noise || !tokens) return invalid("null tensor pointer");
  if (!multiple(logits, dtype == DT_F32 ? 4 : 2) || !multiple(noise, 4)) return invalid("misaligned tensor pointer");
  TcLaunch L;
  const int rc = current_launch(&L);
  if (rc != FPV2_OK) return rc;
  SampleArgs a = {};
  a.logits = logits;
  a.noise = noise;
  a.logits_stride = logits_stride;
  a.noise_stride = noise_stride;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.temperature_s = temperature_all;
  a.top_k_s = top_k_all;
  a.top_p_s = top_p_all;
  a.min_p_s = min_p_all;
  a.rows = (int)rows;
  a.vocab = vocab;
  a.tokens = tokens;
  a.logprobs = logprobs;
  return launched(launch_sample(a, dtype, L.num_sms, reinterpret_cast<cudaStream_t>(stream)),
                  "sample_tokens launch");
}

}  // extern "C"
