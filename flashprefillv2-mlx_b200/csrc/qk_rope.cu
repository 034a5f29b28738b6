// RMS norm of query and key heads, rotary embedding and the write of K and V
// into their cache pages, in one pass.
//
// For a head vector x of D values at position p:
//   y   = x * 1/sqrt(mean(x^2) + eps) * w            (w: per-dimension weight, optional)
//   (a, b) of rotary pair i  ->  (a c_i - b s_i, b c_i + a s_i)
// with c_i, s_i row p of the float32 table (cosines, then sines). Pairs are
// (i, i + rotary/2) or, interleaved, (2i, 2i+1); dimensions past rotary_dim stay
// as normed. All arithmetic is float32, rounded once to the output type.
//
// Every element is read once and written once with a handful of operations, so
// DRAM bandwidth bounds the long calls and launch latency the short ones.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace fpv2 {
namespace {

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i]
              : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// Where head vector `h` of token `t` comes from. Heads are numbered q, then k, then
// (with a cache) v.
__device__ __forceinline__ const char* source_of(const RopeArgs& a, int64_t t, int h, int esize) {
  if (h < a.Hq) return reinterpret_cast<const char*>(a.q) + (t * a.q_st + h * a.q_sh) * esize;
  h -= a.Hq;
  if (h < a.Hkv) return reinterpret_cast<const char*>(a.k) + (t * a.k_st + h * a.k_sh) * esize;
  return reinterpret_cast<const char*>(a.v) + (t * a.v_st + (h - a.Hkv) * a.v_sh) * esize;
}

// Where it goes: null when it is not written (a cache slot out of range).
__device__ __forceinline__ char* target_of(const RopeArgs& a, int64_t t, int h, int64_t slot, int esize) {
  if (h < a.Hq) return reinterpret_cast<char*>(a.q_out) + (t * a.qo_st + h * a.qo_sh) * esize;
  h -= a.Hq;
  if (a.k_cache == nullptr) return reinterpret_cast<char*>(a.k_out) + (t * a.ko_st + h * a.ko_sh) * esize;
  if (slot < 0) return nullptr;
  const int64_t page = slot <= 0x7fffffff ? (uint32_t)slot / (uint32_t)a.page_size : slot / a.page_size;
  const int64_t row = slot - page * a.page_size;
  if (h < a.Hkv)
    return reinterpret_cast<char*>(a.k_cache) + (page * a.kc_sp + row * a.kc_sr + h * a.kc_sh) * esize;
  return reinterpret_cast<char*>(a.v_cache) + (page * a.vc_sp + row * a.vc_sr + (h - a.Hkv) * a.vc_sh) * esize;
}

// Table row of token t: positions outside the table are clamped into it.
__device__ __forceinline__ const float* table_row(const RopeArgs& a, int64_t t) {
  int64_t pos = index_at(a.positions, a.pos64, t);
  pos = pos < 0 ? 0 : (pos >= a.max_pos ? a.max_pos - 1 : pos);
  return a.table + pos * a.rot;
}

// Cache slot of token t, -1 when it is not to be written.
__device__ __forceinline__ int64_t slot_of(const RopeArgs& a, int64_t t) {
  if (a.k_cache == nullptr) return -1;
  const int64_t s = a.slots[t];
  return s >= 0 && s < a.num_slots ? s : -1;
}

// Four values as they are in memory, and as floats.
template <int DT> struct Four;
template <> struct Four<DT_F32> {
  float4 u;
  __device__ __forceinline__ void to(float* x) const { x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w; }
  static __device__ __forceinline__ Four of(const float* x) { return {make_float4(x[0], x[1], x[2], x[3])}; }
};
template <int DT> struct Four {
  uint2 u;
  __device__ __forceinline__ void to(float* x) const {
    const float2 f = unpack2<DT>(u.x), g = unpack2<DT>(u.y);
    x[0] = f.x, x[1] = f.y, x[2] = g.x, x[3] = g.y;
  }
  static __device__ __forceinline__ Four of(const float* x) {
    return {make_uint2(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]))};
  }
};
template <int DT> __device__ __forceinline__ void load4(const void* p, float* x) {
  reinterpret_cast<const Four<DT>*>(p)->to(x);
}

__device__ __forceinline__ void load4_weight(const void* w, int dt, int at, float* x) {
  if (dt == DT_F32)
    load4<DT_F32>(reinterpret_cast<const float*>(w) + at, x);
  else if (dt == DT_BF16)
    load4<DT_BF16>(reinterpret_cast<const uint16_t*>(w) + at, x);
  else
    load4<DT_F16>(reinterpret_cast<const uint16_t*>(w) + at, x);
}

// Vector form: LANES lanes hold one head vector, two fours of it a lane: the two
// sides of four rotary pairs (or four interleaved pairs), so the rotation needs no
// other lane and only four cosines and sines; past rotary_dim, eight in a row. A group
// of LANES lanes takes HPT heads of one token, `apart` heads from one to the next, so
// neighbouring groups read neighbouring heads, the token's table row and cache slot
// are looked up once and HPT heads' loads are in flight.
template <int DT, int LANES, int HPT, bool INTER>
__global__ void __launch_bounds__(256) qk_rope_vec_kernel(const RopeArgs a, int apart) {
  constexpr int ES = DT == DT_F32 ? 4 : 2;
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  const int c = threadIdx.x % LANES;
  const unsigned group = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const unsigned t_raw = group / (unsigned)apart;
  const int h0 = (int)(group - t_raw * apart);
  const bool in = t_raw < a.tokens;    // lanes past the end still take part in shuffles
  const bool live = in && c * 8 < a.D;
  const int64_t t = in ? t_raw : 0;
  const int half = a.rot / 2;
  const bool turns = live && c * 8 < a.rot;
  const int d0 = INTER || c * 8 >= a.rot ? c * 8 : c * 4;
  const int d1 = INTER || c * 8 >= a.rot ? c * 8 + 4 : half + c * 4;

  // strides fit 32 bits here, so an address is one wide multiply-add
  const int kv0 = a.Hq, v0 = a.Hq + a.Hkv;
  const char* qs = reinterpret_cast<const char*>(a.q) + t * (int)a.q_st * ES;
  const char* ks = reinterpret_cast<const char*>(a.k) + t * (int)a.k_st * ES;
  const char* vs = reinterpret_cast<const char*>(a.v) + t * (int)a.v_st * ES;
  const int qsh = (int)a.q_sh * ES, ksh = (int)a.k_sh * ES, vsh = (int)a.v_sh * ES;
  Four<DT> x[HPT][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i * apart;
    x[i][0] = x[i][1] = Four<DT>{};
    if (live && h < heads) {
      const char* src = h < kv0 ? qs + (int64_t)h * qsh
                      : h < v0 ? ks + (int64_t)(h - kv0) * ksh : vs + (int64_t)(h - v0) * vsh;
      x[i][0] = *reinterpret_cast<const Four<DT>*>(src + d0 * ES);
      x[i][1] = *reinterpret_cast<const Four<DT>*>(src + d1 * ES);
    }
  }
  float co[4], si[4];
  if (turns) {
    const float* row = table_row(a, t);
    load4<DT_F32>(row + c * 4, co);
    load4<DT_F32>(row + half + c * 4, si);
  }
  char* const qd = reinterpret_cast<char*>(a.q_out) + t * (int)a.qo_st * ES;
  char *kd, *vd = nullptr;   // null: a cache slot out of range, not written
  int ksd, vsd = 0;
  if (a.k_cache == nullptr) {
    kd = reinterpret_cast<char*>(a.k_out) + t * (int)a.ko_st * ES;
    ksd = (int)a.ko_sh * ES;
  } else {
    const int64_t slot = slot_of(a, t);
    const unsigned page = (unsigned)slot / (unsigned)a.page_size;
    const int row = (int)slot - (int)(page * a.page_size);
    kd = slot < 0 ? nullptr : reinterpret_cast<char*>(a.k_cache) + ((int64_t)page * (int)a.kc_sp + (int64_t)row * (int)a.kc_sr) * ES;
    vd = slot < 0 ? nullptr : reinterpret_cast<char*>(a.v_cache) + ((int64_t)page * (int)a.vc_sp + (int64_t)row * (int)a.vc_sr) * ES;
    ksd = (int)a.kc_sh * ES;
    vsd = (int)a.vc_sh * ES;
  }
  const int qsd = (int)a.qo_sh * ES;
  const float inv_d = 1.f / (float)a.D;
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = h0 + i * apart;
    float y[8];
    x[i][0].to(y);
    x[i][1].to(y + 4);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!live || h >= heads) continue;
    if (h < a.Hq + a.Hkv) {
      const float r = rsqrtf(fmaf(ss, inv_d, a.eps));
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] *= r;
      const void* weight = h < a.Hq ? a.q_weight : a.k_weight;
      if (weight != nullptr) {
        float w[8];
        load4_weight(weight, a.weight_dt, d0, w);
        load4_weight(weight, a.weight_dt, d1, w + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= w[j];
      }
      if (turns) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int p = INTER ? 2 * j : j, q = INTER ? 2 * j + 1 : j + 4;
          const float u = y[p], v = y[q];
          y[p] = u * co[j] - v * si[j];
          y[q] = v * co[j] + u * si[j];
        }
      }
    }
    char* const to = h < kv0 ? qd : h < v0 ? kd : vd;
    if (to != nullptr) {
      char* const dst = to + (h < kv0 ? (int64_t)h * qsd
                              : h < v0 ? (int64_t)(h - kv0) * ksd : (int64_t)(h - v0) * vsd);
      *reinterpret_cast<Four<DT>*>(dst + d0 * ES) = Four<DT>::of(y);
      *reinterpret_cast<Four<DT>*>(dst + d1 * ES) = Four<DT>::of(y + 4);
    }
  }
}

// Any head_dim up to 256, any rotary_dim, any alignment: one warp a head vector,
// values 32 apart in a lane, pairs exchanged through shared memory.
template <int DT>
__global__ void __launch_bounds__(256) qk_rope_any_kernel(const RopeArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ float buf[8][256];
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = (int64_t)blockIdx.x * 8 + warp;
  if (item >= a.tokens * heads) return;
  const int64_t t = item / heads;
  const int h = (int)(item - t * heads);
  const T* src = reinterpret_cast<const T*>(source_of(a, t, h, (int)sizeof(T)));
  T* dst = reinterpret_cast<T*>(target_of(a, t, h, slot_of(a, t), (int)sizeof(T)));
  if (dst == nullptr) return;
  const void* weight = h < a.Hq ? a.q_weight : a.k_weight;
  if (h >= a.Hq + a.Hkv) {
    for (int d = lane; d < a.D; d += 32) dst[d] = src[d];
    return;
  }
  float ss = 0.f;
  for (int d = lane; d < a.D; d += 32) {
    const float x = E::to_f(src[d]);
    buf[warp][d] = x;
    ss = fmaf(x, x, ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = rsqrtf(ss / (float)a.D + a.eps);
  for (int d = lane; d < a.D; d += 32)
    buf[warp][d] *= weight != nullptr ? r * load_as_float(weight, a.weight_dt, d) : r;
  __syncwarp();
  const int half = a.rot / 2;
  const float* row = table_row(a, t);
  for (int d = lane; d < a.D; d += 32) {
    float y = buf[warp][d];
    if (d < a.rot) {
      const int pair = a.interleaved ? d >> 1 : (d < half ? d : d - half);
      const bool first = a.interleaved ? (d & 1) == 0 : d < half;
      const int mate = a.interleaved ? d ^ 1 : (first ? d + half : d - half);
      const float other = buf[warp][mate];
      y = first ? y * row[pair] - other * row[half + pair] : y * row[pair] + other * row[half + pair];
    }
    dst[d] = E::from_f(y);
  }
}

template <int DT, int LANES, int HPT>
cudaError_t launch_vec(const RopeArgs& a, int heads, cudaStream_t stream) {
  const int apart = (heads + HPT - 1) / HPT;
  const int64_t blocks = (a.tokens * apart * LANES + 255) / 256;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (a.interleaved)
    qk_rope_vec_kernel<DT, LANES, HPT, true><<<(unsigned)blocks, 256, 0, stream>>>(a, apart);
  else
    qk_rope_vec_kernel<DT, LANES, HPT, false><<<(unsigned)blocks, 256, 0, stream>>>(a, apart);
  count_launch();
  return cudaGetLastError();
}

template <int DT, int LANES>
cudaError_t launch_vec_heads(const RopeArgs& a, int num_sms, cudaStream_t stream) {
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  // four heads a lane group once that still gives every SM two CTAs
  const bool many = a.tokens * heads * LANES / (256 * 4) >= 2 * num_sms;
  return many ? launch_vec<DT, LANES, 4>(a, heads, stream) : launch_vec<DT, LANES, 1>(a, heads, stream);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int DT> cudaError_t launch_dt(const RopeArgs& a, int num_sms, cudaStream_t stream) {
  constexpr int ES = DT == DT_F32 ? 4 : 2;
  const int64_t strides = a.q_st | a.q_sh | a.k_st | a.k_sh | a.v_st | a.v_sh | a.qo_st | a.qo_sh |
                          a.ko_st | a.ko_sh | a.kc_sp | a.kc_sr | a.kc_sh | a.vc_sp | a.vc_sr | a.vc_sh;
  const bool vec = a.D % 8 == 0 && a.rot % 8 == 0 && (strides * ES) % 16 == 0 &&
                   aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.q_out) &&
                   aligned16(a.k_out) && aligned16(a.k_cache) && aligned16(a.v_cache) &&
                   aligned16(a.table) && aligned16(a.q_weight) && aligned16(a.k_weight);
  // group numbers, slots and strides are 32-bit in the vector kernel
  if (vec && a.tokens * (a.Hq + 2 * a.Hkv) <= 0x7fffffff && a.num_slots <= 0x7fffffff &&
      (strides * ES) >> 31 == 0)
    return a.D <= 64 ? launch_vec_heads<DT, 8>(a, num_sms, stream)
         : a.D <= 128 ? launch_vec_heads<DT, 16>(a, num_sms, stream)
                      : launch_vec_heads<DT, 32>(a, num_sms, stream);
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  const int64_t blocks = (a.tokens * heads + 7) / 8;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  qk_rope_any_kernel<DT><<<(unsigned)blocks, 256, 0, stream>>>(a);
  count_launch();
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_qk_rope(const RopeArgs& a, int dt, int num_sms, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  if (dt == DT_BF16) return launch_dt<DT_BF16>(a, num_sms, stream);
  if (dt == DT_F16) return launch_dt<DT_F16>(a, num_sms, stream);
  return launch_dt<DT_F32>(a, num_sms, stream);
}

}  // namespace fpv2
