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
#include "common.cuh"
#include "kernels.h"

namespace fpv2 {
namespace {

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i]
              : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// Where head vector `h` of token `t` comes from and goes to. Heads are numbered
// q, then k, then (with a cache) v. A null destination means the vector is not
// written (a cache slot out of range: padding tokens).
struct VecPlace {
  const char* src;
  char* dst;
  const void* weight;
  bool rotate;
};

__device__ __forceinline__ VecPlace place_of(const RopeArgs& a, int64_t t, int h, int64_t slot,
                                             int esize) {
  VecPlace p;
  if (h < a.Hq) {
    p.src = reinterpret_cast<const char*>(a.q) + (t * a.q_st + (int64_t)h * a.q_sh) * esize;
    p.dst = reinterpret_cast<char*>(a.q_out) + (t * a.qo_st + (int64_t)h * a.qo_sh) * esize;
    p.weight = a.q_weight;
    p.rotate = true;
    return p;
  }
  h -= a.Hq;
  const bool is_k = h < a.Hkv;
  if (!is_k) h -= a.Hkv;
  p.src = is_k ? reinterpret_cast<const char*>(a.k) + (t * a.k_st + (int64_t)h * a.k_sh) * esize
               : reinterpret_cast<const char*>(a.v) + (t * a.v_st + (int64_t)h * a.v_sh) * esize;
  p.weight = is_k ? a.k_weight : nullptr;
  p.rotate = is_k;
  if (a.k_cache == nullptr) {
    p.dst = reinterpret_cast<char*>(a.k_out) + (t * a.ko_st + (int64_t)h * a.ko_sh) * esize;
  } else if (slot < 0) {
    p.dst = nullptr;
  } else {
    const int64_t page = slot / a.page_size, row = slot - page * a.page_size;
    p.dst = is_k ? reinterpret_cast<char*>(a.k_cache) +
                       (page * a.kc_sp + row * a.kc_sr + (int64_t)h * a.kc_sh) * esize
                 : reinterpret_cast<char*>(a.v_cache) +
                       (page * a.vc_sp + row * a.vc_sr + (int64_t)h * a.vc_sh) * esize;
  }
  return p;
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

template <int DT> __device__ __forceinline__ void load8(const void* p, float (&x)[8]) {
  if constexpr (DT == DT_F32) {
    const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
    x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<DT>(r[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

template <int DT> __device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
  if constexpr (DT == DT_F32) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]),
                                              pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7]));
  }
}

__device__ __forceinline__ void load8_weight(const void* w, int dt, int at, float (&x)[8]) {
  if (dt == DT_F32)
    load8<DT_F32>(reinterpret_cast<const float*>(w) + at, x);
  else if (dt == DT_BF16)
    load8<DT_BF16>(reinterpret_cast<const uint16_t*>(w) + at, x);
  else
    load8<DT_F16>(reinterpret_cast<const uint16_t*>(w) + at, x);
}

// Vector form: LANES lanes hold one head vector, eight values a lane, and take
// HPT heads of the same token, whose table row they load once.
template <int DT, int LANES, int HPT, bool INTER>
__global__ void __launch_bounds__(256) qk_rope_vec_kernel(const RopeArgs a) {
  constexpr int ES = DT == DT_F32 ? 4 : 2;
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  const int blocks_per_token = (heads + HPT - 1) / HPT;
  const int64_t group = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LANES;
  const int c = threadIdx.x % LANES;                 // this lane's chunk of eight values
  const int64_t t_raw = group / blocks_per_token;
  const int h0 = (int)(group - t_raw * blocks_per_token) * HPT;
  const bool live = t_raw < a.tokens && c * 8 < a.D;   // lanes past the end still take part in shuffles
  const int64_t t = t_raw < a.tokens ? t_raw : a.tokens - 1;

  float x[HPT][8];
  VecPlace pl[HPT];
  const int64_t slot = slot_of(a, t);
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = min(h0 + i, heads - 1);
    pl[i] = place_of(a, t, h, slot, ES);
    if (live) {
      load8<DT>(pl[i].src + c * 8 * ES, x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
    }
  }
  const int half = a.rot / 2;
  const bool turns = live && c * 8 < a.rot;
  float co[8], si[8];   // interleaved: four pairs, each value twice in effect
  if (turns) {
    const float* row = table_row(a, t);
    if constexpr (INTER) {
      const float4 cc = *reinterpret_cast<const float4*>(row + c * 4);
      const float4 ss = *reinterpret_cast<const float4*>(row + half + c * 4);
      co[0] = cc.x, co[1] = cc.y, co[2] = cc.z, co[3] = cc.w;
      si[0] = ss.x, si[1] = ss.y, si[2] = ss.z, si[3] = ss.w;
    } else {
      const int at = c * 8 < half ? c * 8 : c * 8 - half;
      load8<DT_F32>(row + at, co);
      load8<DT_F32>(row + half + at, si);
    }
  }
  const int lane = threadIdx.x & 31;
  const bool first_half = c * 8 < half;
  const int partner = turns ? lane + (first_half ? half / 8 : -half / 8) : lane;
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[i][j], x[i][j], ss);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    float y[8];
    if (pl[i].rotate) {
      const float r = rsqrtf(ss / (float)a.D + a.eps);
      if (pl[i].weight != nullptr && live) {
        float w[8];
        load8_weight(pl[i].weight, a.weight_dt, c * 8, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[i][j] * r * w[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[i][j] * r;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = x[i][j];
    }
    if constexpr (INTER) {
      if (turns && pl[i].rotate) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = y[2 * j], v = y[2 * j + 1];
          y[2 * j] = u * co[j] - v * si[j];
          y[2 * j + 1] = v * co[j] + u * si[j];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float other = __shfl_sync(0xffffffffu, y[j], partner);
        if (turns && pl[i].rotate)
          y[j] = first_half ? y[j] * co[j] - other * si[j] : y[j] * co[j] + other * si[j];
      }
    }
    if (live && h0 + i < heads && pl[i].dst != nullptr) store8<DT>(pl[i].dst + c * 8 * ES, y);
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
  const VecPlace pl = place_of(a, t, h, slot_of(a, t), (int)sizeof(T));
  const T* src = reinterpret_cast<const T*>(pl.src);
  T* dst = reinterpret_cast<T*>(pl.dst);
  if (dst == nullptr) return;
  if (!pl.rotate) {
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
    buf[warp][d] *= pl.weight != nullptr ? r * load_as_float(pl.weight, a.weight_dt, d) : r;
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
void launch_vec(const RopeArgs& a, int64_t blocks, cudaStream_t stream) {
  if (a.interleaved)
    qk_rope_vec_kernel<DT, LANES, HPT, true><<<(unsigned)blocks, 256, 0, stream>>>(a);
  else
    qk_rope_vec_kernel<DT, LANES, HPT, false><<<(unsigned)blocks, 256, 0, stream>>>(a);
}

template <int DT, int HPT>
cudaError_t launch_vec_lanes(const RopeArgs& a, cudaStream_t stream) {
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  const int lanes = a.D <= 64 ? 8 : a.D <= 128 ? 16 : 32;
  const int64_t groups = a.tokens * ((heads + HPT - 1) / HPT);
  const int64_t blocks = (groups * lanes + 255) / 256;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (lanes == 8)
    launch_vec<DT, 8, HPT>(a, blocks, stream);
  else if (lanes == 16)
    launch_vec<DT, 16, HPT>(a, blocks, stream);
  else
    launch_vec<DT, 32, HPT>(a, blocks, stream);
  count_launch();
  return cudaGetLastError();
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int DT> cudaError_t launch_dt(const RopeArgs& a, int num_sms, cudaStream_t stream) {
  constexpr int ES = DT == DT_F32 ? 4 : 2;
  const int64_t strides = a.q_st | a.q_sh | a.k_st | a.k_sh | a.v_st | a.v_sh | a.qo_st | a.qo_sh |
                          a.ko_st | a.ko_sh | a.kc_sp | a.kc_sr | a.kc_sh | a.vc_sp | a.vc_sr | a.vc_sh;
  const bool vec = a.D % 8 == 0 && a.rot % (a.interleaved ? 8 : 16) == 0 && (strides * ES) % 16 == 0 &&
                   aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.q_out) &&
                   aligned16(a.k_out) && aligned16(a.k_cache) && aligned16(a.v_cache) &&
                   aligned16(a.table) && aligned16(a.q_weight) && aligned16(a.k_weight);
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  if (vec) {
    (void)num_sms;
    return launch_vec_lanes<DT, 1>(a, stream);
  }
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
