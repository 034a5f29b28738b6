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
#include <cstdint>

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

__device__ __forceinline__ float2 mul_f32x2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// BYTES (8 or 16) of values as they are in memory, and as pairs of floats.
template <int DT, int BYTES> struct Pack {
  static constexpr int N = BYTES / (DT == DT_F32 ? 4 : 2), WORDS = BYTES / 4;
  uint32_t u[WORDS];
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (BYTES == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      u[0] = v.x, u[1] = v.y, u[2] = v.z, u[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      u[0] = v.x, u[1] = v.y;
    }
  }
  __device__ __forceinline__ void store(void* p) const {
    if constexpr (BYTES == 16)
      *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    else
      *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
  }
  __device__ __forceinline__ void to(float2* x) const {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (DT == DT_F32)
        x[i] = make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
      else
        x[i] = unpack2<DT>(u[i]);
    }
  }
  __device__ __forceinline__ void from(const float2* x) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (DT == DT_F32) {
        u[2 * i] = __float_as_uint(x[i].x);
        u[2 * i + 1] = __float_as_uint(x[i].y);
      } else {
        u[i] = pack2<DT>(x[i].x, x[i].y);
      }
    }
  }
};
template <int BYTES> __device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}

// N floats as pairs
template <int N> __device__ __forceinline__ void load_floats(const float* p, float2* x) {
  if constexpr (N == 2) {
    x[0] = *reinterpret_cast<const float2*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i / 2] = make_float2(v.x, v.y);
      x[i / 2 + 1] = make_float2(v.z, v.w);
    }
  }
}
template <int N> __device__ __forceinline__ void load_weights(const void* w, int dt, int at, float2* x) {
  if (dt == DT_F32) {
    load_floats<N>(reinterpret_cast<const float*>(w) + at, x);
  } else if (dt == DT_BF16) {
    Pack<DT_BF16, 2 * N> p;
    p.load(reinterpret_cast<const uint16_t*>(w) + at);
    p.to(x);
  } else {
    Pack<DT_F16, 2 * N> p;
    p.load(reinterpret_cast<const uint16_t*>(w) + at);
    p.to(x);
  }
}

// Vector form: LANES lanes hold one head vector, two packs of it a lane, so neighbouring
// lanes read neighbouring packs: the two sides of N rotary pairs (or N interleaved
// pairs), so the rotation needs no other lane. A group of LANES lanes takes heads of one
// token, `apart` heads from one to the next, so neighbouring groups read neighbouring
// heads, the token's table row and cache slot are looked up once and the norm weights
// stay in registers from head to head.
//
// DRAM bounds it once enough is on its way: the next AHEAD heads are copied to shared
// memory meanwhile, where they cost no registers (held in registers, two ahead, 16384
// bf16 tokens of 32 + 8 + 8 heads of 128 took 97 us, half of a warp's time waiting for
// loads; so 72 us, 5.7 TB/s; float32, 32 + 8 heads: 115 and 105 us, 6.5 TB/s, a copy's
// rate). 5 ahead measure the same as 3. Two CTAs of 256 threads an SM hold a 16-bit type's
// values without spills (4096 tokens 19.6 us; three CTAs 23.5 us), four a float32 type's,
// which are half as many a lane. With AHEAD 0 a group takes one head (few tokens),
// loaded to registers.
template <int DT, int AHEAD> constexpr int kCtas = AHEAD == 0 ? 3 : DT == DT_F32 ? 4 : 2;

template <int DT, int BYTES, int LANES, bool INTER, int AHEAD>
__global__ void __launch_bounds__(256, (kCtas<DT, AHEAD>)) qk_rope_vec_kernel(const RopeArgs a, int apart) {
  using P = Pack<DT, BYTES>;
  constexpr int ES = DT == DT_F32 ? 4 : 2, N = P::N, H = N / 2;
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  const int c = threadIdx.x % LANES;
  const unsigned group = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const unsigned t_raw = group / (unsigned)apart;
  const int h0 = (int)(group - t_raw * apart);
  const bool in = t_raw < a.tokens;    // lanes past the end still take part in shuffles
  const bool live = in && c * 2 * N < a.D;
  const int64_t t = in ? t_raw : 0;
  // the dimensions of the lane's two packs, and what of them is rotated
  const int half = a.rot / 2, rest = a.D - a.rot;
  int d0, d1;
  bool turn0, turn1;
  if (INTER) {
    d0 = c * N;
    d1 = a.D / 2 + c * N;
    turn0 = live && d0 < a.rot;
    turn1 = live && d1 < a.rot;
  } else {
    turn0 = turn1 = live && c * N < half;
    d0 = c * N < half ? c * N : a.rot + c * N - half;
    d1 = c * N < half ? half + c * N : d0 + rest / 2;
  }

  // strides fit 32 bits here, so an address is one wide multiply-add
  const int kv0 = a.Hq, v0 = a.Hq + a.Hkv;
  const char* qs = reinterpret_cast<const char*>(a.q) + t * (int)a.q_st * ES;
  const char* ks = reinterpret_cast<const char*>(a.k) + t * (int)a.k_st * ES;
  const char* vs = reinterpret_cast<const char*>(a.v) + t * (int)a.v_st * ES;
  const int qsh = (int)a.q_sh * ES, ksh = (int)a.k_sh * ES, vsh = (int)a.v_sh * ES;
  auto source = [&](int h) {
    return h < kv0 ? qs + (int64_t)h * qsh
         : h < v0 ? ks + (int64_t)(h - kv0) * ksh : vs + (int64_t)(h - v0) * vsh;
  };
  // the heads on their way, each lane's own two packs: no lane reads another's, so a wait
  // for the lane's copies is all the order they need
  __shared__ __align__(16) unsigned char ring[AHEAD > 0 ? (AHEAD + 1) * 2 * 256 * BYTES : 16];
  const uint32_t mine_at = smem_u32(ring) + threadIdx.x * BYTES;
  P mine[2] = {};
  auto issue = [&](int h, int slot) {
    if (live && h < heads) {
      const char* src = source(h);
      cp_async<BYTES>(mine_at + slot * 2 * 256 * BYTES, src + d0 * ES);
      cp_async<BYTES>(mine_at + (slot * 2 + 1) * 256 * BYTES, src + d1 * ES);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (AHEAD > 0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) issue(h0 + i * apart, i);
  } else if (live && h0 < heads) {
    const char* src = source(h0);
    mine[0].load(src + d0 * ES);
    mine[1].load(src + d1 * ES);
  }
  float2 co[H], si[H];   // interleaved: of the first pack's pairs, then of the second's
#pragma unroll
  for (int j = 0; j < H; ++j) {   // no rotation: by nothing
    co[j] = make_float2(1.f, 1.f);
    si[j] = make_float2(0.f, 0.f);
  }
  const float* row = table_row(a, t);
  if constexpr (INTER) {
    if (turn0) {
      load_floats<H>(row + d0 / 2, co);
      load_floats<H>(row + half + d0 / 2, si);
    }
    if (turn1) {
      load_floats<H>(row + d1 / 2, co + H / 2);
      load_floats<H>(row + half + d1 / 2, si + H / 2);
    }
  } else if (turn0) {
    load_floats<N>(row + c * N, co);
    load_floats<N>(row + half + c * N, si);
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
    const int in_page = (int)slot - (int)(page * a.page_size);
    kd = slot < 0 ? nullptr : reinterpret_cast<char*>(a.k_cache) + ((int64_t)page * (int)a.kc_sp + (int64_t)in_page * (int)a.kc_sr) * ES;
    vd = slot < 0 ? nullptr : reinterpret_cast<char*>(a.v_cache) + ((int64_t)page * (int)a.vc_sp + (int64_t)in_page * (int)a.vc_sr) * ES;
    ksd = (int)a.kc_sh * ES;
    vsd = (int)a.vc_sh * ES;
  }
  const int qsd = (int)a.qo_sh * ES;
  const float inv_d = 1.f / (float)a.D;
  const void* have = nullptr;
  float2 w[2 * H];
#pragma unroll
  for (int j = 0; j < 2 * H; ++j) w[j] = make_float2(1.f, 1.f);
  float2 ns[H];   // the sines, negated
#pragma unroll
  for (int j = 0; j < H; ++j) ns[j] = make_float2(-si[j].x, -si[j].y);
  // every lane of a warp takes the same number of steps
  const int steps = (heads + apart - 1) / apart;
  int slot = 0, fill = AHEAD;
  for (int step = 0, h = h0; step < steps; ++step, h += apart) {
    if constexpr (AHEAD > 0) {
      issue(h + AHEAD * apart, fill);
      fill = slot;
      asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
      if (live) {   // the other lanes' values stay 0, for the sum of squares
        mine[0].load(ring + slot * 2 * 256 * BYTES + threadIdx.x * BYTES);
        mine[1].load(ring + (slot * 2 + 1) * 256 * BYTES + threadIdx.x * BYTES);
      }
      slot = slot == AHEAD ? 0 : slot + 1;
    }
    float2 y[2 * H];
    mine[0].to(y);
    mine[1].to(y + H);
    float2 s2 = mul_f32x2(y[0], y[0]);
#pragma unroll
    for (int j = 1; j < 2 * H; ++j) s2 = fma_f32x2(y[j], y[j], s2);
    float ss = s2.x + s2.y;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    char* const to = h < kv0 ? qd : h < v0 ? kd : vd;
    if (!live || h >= heads || to == nullptr) continue;
    char* const dst = to + (h < kv0 ? (int64_t)h * qsd
                            : h < v0 ? (int64_t)(h - kv0) * ksd : (int64_t)(h - v0) * vsd);
    if (h < v0) {
      const float r = rsqrtf(fmaf(ss, inv_d, a.eps));
      const void* weight = h < kv0 ? a.q_weight : a.k_weight;
      if (weight != have) {
        have = weight;
        if (weight != nullptr) {
          load_weights<N>(weight, a.weight_dt, d0, w);
          load_weights<N>(weight, a.weight_dt, d1, w + H);
        } else {
#pragma unroll
          for (int j = 0; j < 2 * H; ++j) w[j] = make_float2(1.f, 1.f);
        }
      }
#pragma unroll
      for (int j = 0; j < 2 * H; ++j) y[j] = mul_f32x2(mul_f32x2(y[j], make_float2(r, r)), w[j]);
      if constexpr (INTER) {
#pragma unroll
        for (int j = 0; j < 2 * H; ++j) {
          const float cj = j & 1 ? co[j / 2].y : co[j / 2].x;
          const float sj = j & 1 ? si[j / 2].y : si[j / 2].x, nj = j & 1 ? ns[j / 2].y : ns[j / 2].x;
          y[j] = fma_f32x2(y[j], make_float2(cj, cj), mul_f32x2(make_float2(y[j].y, y[j].x), make_float2(nj, sj)));
        }
      } else {
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const float2 p = y[j], v = y[j + H];
          y[j] = fma_f32x2(p, co[j], mul_f32x2(v, ns[j]));
          y[j + H] = fma_f32x2(v, co[j], mul_f32x2(p, si[j]));
        }
      }
      mine[0].from(y);
      mine[1].from(y + H);
    }
    mine[0].store(dst + d0 * ES);
    mine[1].store(dst + d1 * ES);
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

template <int DT, int BYTES, int LANES, int AHEAD>
cudaError_t launch_apart(const RopeArgs& a, int apart, cudaStream_t stream) {
  const int64_t blocks = (a.tokens * apart * LANES + 255) / 256;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (a.interleaved)
    qk_rope_vec_kernel<DT, BYTES, LANES, true, AHEAD><<<(unsigned)blocks, 256, 0, stream>>>(a, apart);
  else
    qk_rope_vec_kernel<DT, BYTES, LANES, false, AHEAD><<<(unsigned)blocks, 256, 0, stream>>>(a, apart);
  count_launch();
  return cudaGetLastError();
}

template <int DT, int BYTES, int LANES>
cudaError_t launch_lanes(const RopeArgs& a, int num_sms, cudaStream_t stream) {
  constexpr int AHEAD = 3;
  const int heads = a.Hq + (a.k_cache != nullptr ? 2 : 1) * a.Hkv;
  constexpr int GROUPS = 256 / LANES;   // of a CTA
  // one head a lane group while the CTAs about fit on the GPU at once
  if (a.tokens * heads <= 4ll * num_sms * GROUPS)
    return launch_apart<DT, BYTES, LANES, 0>(a, heads, stream);
  // else as many as make the shortest sum of waves of CTAs, a group's start (its token's
  // table row, the weights) counting as three heads (31007 tokens of 16 + 4
  // float32 heads of 96: 76 us; by the CTAs an SM gets, which evens out part waves, 82 us)
  const int64_t slots = (int64_t)kCtas<DT, AHEAD> * num_sms * GROUPS;
  int best = heads;
  int64_t least = INT64_MAX;
  for (int steps = 1; steps <= std::min(heads, 24); ++steps) {
    const int apart = (heads + steps - 1) / steps;
    const int64_t cost = (a.tokens * apart + slots - 1) / slots * (steps + 3);
    if (cost < least) {
      least = cost;
      best = apart;
    }
  }
  return launch_apart<DT, BYTES, LANES, AHEAD>(a, best, stream);
}

template <int DT, int BYTES> cudaError_t launch_vec(const RopeArgs& a, int num_sms, cudaStream_t stream) {
  constexpr int PER = 2 * Pack<DT, BYTES>::N;   // values a lane
  return a.D <= 64 ? launch_lanes<DT, BYTES, 64 / PER>(a, num_sms, stream)
       : a.D <= 128 ? launch_lanes<DT, BYTES, 128 / PER>(a, num_sms, stream)
                    : launch_lanes<DT, BYTES, 256 / PER>(a, num_sms, stream);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int DT> cudaError_t launch_dt(const RopeArgs& a, int num_sms, cudaStream_t stream) {
  constexpr int ES = DT == DT_F32 ? 4 : 2;
  const int64_t strides = a.q_st | a.q_sh | a.k_st | a.k_sh | a.v_st | a.v_sh | a.qo_st | a.qo_sh |
                          a.ko_st | a.ko_sh | a.kc_sp | a.kc_sr | a.kc_sh | a.vc_sp | a.vc_sr | a.vc_sh;
  const bool vec = (strides * ES) % 16 == 0 && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) &&
                   aligned16(a.q_out) && aligned16(a.k_out) && aligned16(a.k_cache) &&
                   aligned16(a.v_cache) && aligned16(a.table) && aligned16(a.q_weight) &&
                   aligned16(a.k_weight) &&
                   // group numbers, slots and strides are 32-bit in the vector kernel
                   a.tokens * (a.Hq + 2 * a.Hkv) <= 0x7fffffff && a.num_slots <= 0x7fffffff &&
                   (strides * ES) >> 31 == 0;
  // whole packs on each side of a rotary pair and past the rotated part
  auto packs = [&](int n) { return a.rot % (2 * n) == 0 && (a.D - a.rot) % (2 * n) == 0; };
  if (vec && packs(16 / ES)) return launch_vec<DT, 16>(a, num_sms, stream);
  if constexpr (DT != DT_F32)
    if (vec && packs(8 / ES)) return launch_vec<DT, 8>(a, num_sms, stream);
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
