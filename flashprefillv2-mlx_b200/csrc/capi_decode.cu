// C ABI of the decode step (declared in include/fpv2_b200.h): argument checks
// and launches, as in capi.cu.
#include <algorithm>
#include <cfloat>
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

constexpr int64_t kMaxSize = 0x7fffffff;
constexpr int64_t kMaxRows = 1 << 24;   // query rows a sequence

bool multiple(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace fpv2

using namespace fpv2;

extern "C" {

int fpv2_qk_norm_rope(const fpv2_qk_norm_rope_params* p, void* stream) {
  if (!p) return invalid("null parameters");
  if (p->dtype != DT_F16 && p->dtype != DT_BF16 && p->dtype != DT_F32) return invalid("unknown dtype code");
  if ((p->q_weight || p->k_weight) && p->weight_dtype != DT_F16 && p->weight_dtype != DT_BF16 &&
      p->weight_dtype != DT_F32)
    return invalid("unknown weight dtype code");
  if (p->tokens < 0 || p->q_heads <= 0 || p->kv_heads <= 0 || p->q_heads > kMaxSize || p->kv_heads > kMaxSize ||
      p->tokens > kMaxSize)
    return invalid("invalid shape");
  if (p->head_dim <= 0 || p->head_dim > 256) return invalid("head dimension must be in [1, 256]");
  if (p->rotary_dim <= 0 || p->rotary_dim % 2 || p->rotary_dim > p->head_dim)
    return invalid("rotary_dim must be even and in [2, head_dim]");
  if (p->table_positions <= 0) return invalid("the rotation table is empty");
  if (!(p->eps >= 0.0 && p->eps <= FLT_MAX)) return invalid("eps must be non-negative and finite in float32");
  const bool paged = p->k_cache != nullptr || p->v_cache != nullptr;
  if (paged && (!p->k_cache || !p->v_cache || !p->slots || p->num_pages <= 0 || p->page_size <= 0 ||
                p->page_size > kMaxSize))
    return invalid("a cache needs k and v pages, a page size and slots");
  if (p->tokens == 0) return FPV2_OK;
  if (!p->q || !p->k || !p->positions || !p->table || !p->q_out || (paged ? !p->v : !p->k_out))
    return invalid("null tensor pointer");
  TcLaunch L;
  const int rc = current_launch(&L);
  if (rc != FPV2_OK) return rc;
  RopeArgs a = {};
  a.q = p->q;
  a.k = p->k;
  a.q_st = p->q_token_stride;
  a.q_sh = p->q_head_stride;
  a.k_st = p->k_token_stride;
  a.k_sh = p->k_head_stride;
  a.positions = p->positions;
  a.pos64 = p->positions_int64 ? 1 : 0;
  a.table = p->table;
  a.max_pos = p->table_positions;
  a.rot = (int)p->rotary_dim;
  a.interleaved = p->interleaved ? 1 : 0;
  a.q_weight = p->q_weight;
  a.k_weight = p->k_weight;
  a.weight_dt = (int)p->weight_dtype;
  a.eps = p->eps > 0.0 ? std::max((float)p->eps, FLT_TRUE_MIN) : 0.f;   // a row of zeros stays one of zeros
  a.q_out = p->q_out;
  a.qo_st = p->q_out_token_stride;
  a.qo_sh = p->q_out_head_stride;
  if (paged) {
    a.v = p->v;
    a.v_st = p->v_token_stride;
    a.v_sh = p->v_head_stride;
    a.k_cache = p->k_cache;
    a.v_cache = p->v_cache;
    a.kc_sp = p->k_page_stride;
    a.kc_sr = p->k_row_stride;
    a.kc_sh = p->k_cache_head_stride;
    a.vc_sp = p->v_page_stride;
    a.vc_sr = p->v_row_stride;
    a.vc_sh = p->v_cache_head_stride;
    a.slots = p->slots;
    a.page_size = (int)p->page_size;
    a.num_slots = p->num_pages * p->page_size;
  } else {
    a.k_out = p->k_out;
    a.ko_st = p->k_out_token_stride;
    a.ko_sh = p->k_out_head_stride;
  }
  a.tokens = p->tokens;
  a.Hq = (int)p->q_heads;
  a.Hkv = (int)p->kv_heads;
  a.D = (int)p->head_dim;
  return launched(launch_qk_rope(a, (int)p->dtype, L.num_sms, reinterpret_cast<cudaStream_t>(stream)),
                  "qk_norm_rope launch");
}

int64_t fpv2_decode_workspace_bytes(int32_t new_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (new_tokens <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || !decode_supported(head_dim) ||
      (int64_t)q_heads * new_tokens > kMaxRows)
    return 0;
  return (int64_t)decode_workspace_bytes(new_tokens, q_heads, kv_heads, head_dim);
}

int fpv2_decode_attention(const fpv2_decode_attention_params* p, void* stream) {
  if (!p) return invalid("null parameters");
  if (p->dtype != DT_F16 && p->dtype != DT_BF16)
    return invalid("q and the caches must share float16 or bfloat16 dtype");
  if (p->batch < 0 || p->batch > kMaxSize || p->new_tokens <= 0 || p->new_tokens > kMaxRows)
    return invalid("invalid shape");
  if (p->kv_heads <= 0 || p->q_heads <= 0 || p->q_heads > kMaxRows || p->q_heads % p->kv_heads)
    return invalid("query heads must be divisible by KV heads");
  if (p->q_heads * p->new_tokens > kMaxRows) return invalid("too many query rows a sequence");
  if (p->head_dim > 256 || !decode_supported((int)p->head_dim))
    return invalid("head dimension must be 64, 96, 128 or 256");
  if (p->num_pages <= 0 || p->page_size <= 0 || p->table_width <= 0 || p->num_pages > kMaxSize ||
      p->page_size > kMaxSize || p->table_width > kMaxSize)
    return invalid("paged K/V needs block tables, pages and a page size");
  if (p->table_width * p->page_size > 0x7fffffff - 64) return invalid("sequences must be shorter than 2^31 keys");
  if (p->window < 0 || p->sinks < 0 || p->window > kMaxSize || p->sinks > kMaxSize)
    return invalid("window and sinks must be non-negative 32-bit integers");
  if (!(std::fabs(p->scale) * kLog2e <= FLT_MAX)) return invalid("scale must be finite, as its product with log2(e) in float32");
  if (p->batch == 0) return FPV2_OK;
  if (!p->q || !p->k_pages || !p->v_pages || !p->block_tables || !p->lengths || !p->out || !p->workspace)
    return invalid("null tensor pointer");
  if (!multiple(p->workspace, 16) ||
      p->workspace_bytes < (int64_t)decode_workspace_bytes((int)p->new_tokens, (int)p->q_heads,
                                                           (int)p->kv_heads, (int)p->head_dim))
    return invalid("workspace is too small or not 16-byte aligned");
  if ((p->q_batch_stride | p->q_token_stride | p->q_head_stride) % 2 ||
      (p->k_page_stride | p->k_row_stride | p->k_head_stride | p->v_page_stride | p->v_row_stride |
       p->v_head_stride) % 8)
    return invalid("q strides must be multiples of 2 elements, cache strides of 8");
  if (!multiple(p->q, 4) || !multiple(p->out, 4) || !multiple(p->k_pages, 16) || !multiple(p->v_pages, 16))
    return invalid("q and out must be 4-byte aligned, the caches 16-byte");
  TcLaunch L;
  const int rc = current_launch(&L);
  if (rc != FPV2_OK) return rc;
  DecodeArgs a = {};
  a.q = p->q;
  a.k = p->k_pages;
  a.v = p->v_pages;
  a.q_sb = p->q_batch_stride;
  a.q_st = p->q_token_stride;
  a.q_sh = p->q_head_stride;
  a.k_sp = p->k_page_stride;
  a.k_sr = p->k_row_stride;
  a.k_sh = p->k_head_stride;
  a.v_sp = p->v_page_stride;
  a.v_sr = p->v_row_stride;
  a.v_sh = p->v_head_stride;
  a.tables = p->block_tables;
  a.lengths = p->lengths;
  a.table_stride = p->table_stride;
  a.B = (int)p->batch;
  a.T = (int)p->new_tokens;
  a.Hq = (int)p->q_heads;
  a.Hkv = (int)p->kv_heads;
  a.G = a.Hq / a.Hkv;
  a.D = (int)p->head_dim;
  a.num_pages = (int)p->num_pages;
  a.page_size = (int)p->page_size;
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a.page_size == 1 << i) a.page_shift = i;
  a.table_width = (int)p->table_width;
  a.window = (int)p->window;
  a.sinks = (int)p->sinks;
  a.scale_log2 = (float)p->scale * kLog2e;
  a.out = p->out;
  a.lse = p->lse;
  a.workspace = p->workspace;
  a.status = L.status;
  return launched(launch_decode(a, (int)p->dtype, reinterpret_cast<cudaStream_t>(stream)),
                  "decode_attention launch");
}

int fpv2_sample_tokens(const fpv2_sample_tokens_params* p, void* stream) {
  if (!p) return invalid("null parameters");
  if (p->dtype != DT_F16 && p->dtype != DT_BF16 && p->dtype != DT_F32) return invalid("unknown dtype code");
  if (p->rows < 0 || p->rows > (1 << 24) || p->vocab <= 0 || p->vocab > (1 << 30)) return invalid("invalid shape");
  if (p->rows == 0) return FPV2_OK;
  if (!p->logits || !p->noise || !p->tokens) return invalid("null tensor pointer");
  if (!multiple(p->logits, p->dtype == DT_F32 ? 4 : 2) || !multiple(p->noise, 4))
    return invalid("misaligned tensor pointer");
  TcLaunch L;
  const int rc = current_launch(&L);
  if (rc != FPV2_OK) return rc;
  SampleArgs a = {};
  a.logits = p->logits;
  a.noise = p->noise;
  a.logits_stride = p->logits_stride;
  a.noise_stride = p->noise_stride;
  a.temperature = p->temperature;
  a.top_k = p->top_k;
  a.top_p = p->top_p;
  a.min_p = p->min_p;
  a.temperature_s = (float)p->temperature_all;
  a.top_k_s = (int)std::min<int64_t>(std::max<int64_t>(p->top_k_all, 0), 0x7fffffff);
  a.top_p_s = (float)p->top_p_all;
  a.min_p_s = (float)p->min_p_all;
  a.rows = (int)p->rows;
  a.vocab = (int)p->vocab;
  a.tokens = p->tokens;
  a.logprobs = p->logprobs;
  return launched(launch_sample(a, (int)p->dtype, L.num_sms, reinterpret_cast<cudaStream_t>(stream)),
                  "sample_tokens launch");
}

}  // extern "C"
