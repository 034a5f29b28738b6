// The next token of each row of logits, from given exponential random numbers.
//
// With x the logits (NaN counts as -inf), z = (x - max)/T and w = e^z, tokens are
// ordered by (x descending, index ascending) and filtered in turn:
//   top-k   the first k
//   top-p   the shortest prefix of those whose weight reaches p times their weight
//   min-p   those with w >= min_p (the first token always stays)
// and the token is argmax(z - log e) over what is left, ties to the lowest index:
// for e ~ Exp(1) a draw with probabilities w / sum w. T <= 0 takes the lowest index
// of the maximum. A row without a logit above -inf gives -1.
//
// A row is read from DRAM once by a cluster of 1 to 8 CTAs: streamed where nothing filters it,
// else into shared memory, with noise read only where a token is still in the running. The
// bytes of the two bound large batches and the chain of cluster-wide steps single rows.
//
// Nothing is sorted but short lists. Top-k: every thread knows the largest logit of
// its share; the (k / CTAs)-th largest of a CTA's 512 such values is a bound that at
// least k logits reach, and hardly more, so the few logits past it are gathered and
// sorted. Top-p alone: logits are counted in 1024 bins linear in x over the part below the
// maximum where the prefix can end; the two bins around the place where the weight crosses
// p of it are gathered and sorted, and the weight above them summed. Where such a list would not
// hold the candidates (very large k, very many equal logits) the threshold is found by
// counting alone, over the ordered bit patterns inside the crossing bin until it holds
// one value. Counts are integers and sums run in a fixed order, so a call repeats bit
// for bit.
//
// Measured, 151936 logits a row: one bf16 row, top-k 50 and top-p, 8.4 us; 64 float32 rows, top-p,
// with log-probabilities 73 us; 200 bf16 rows unfiltered, with log-probabilities 45 us, 4.1 TB/s of
// logits and noise, their largest alone 18 us. 33 float16 rows of 50003 under every filter 19.9 us.
// Found by counting (float32, top-k 9000 and top-p): one row 56 us, 64 rows 151 us.
#include <algorithm>

#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace fpv2 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2 * kThreads;          // of the linear histogram, two a thread
constexpr int kKeyBits = 9;                  // bins over bit patterns, one a thread
constexpr int kList = 2048;                  // gathered candidates of a row
constexpr int kFew = kThreads / 2;           // of them that one CTA looks through by itself
constexpr int kListBytes = kList * 12;       // keys with indices, and weights
// Logits a CTA holds when two share an SM (200 rows of 151936 bf16, unfiltered, and the nucleus
// of 64 float32 rows: 51.6 and 73.0 us; a cap of 40 KB 71.2 and 73.1, of 160 KB 65.7 and 79.2), and
// when it has the SM to itself
constexpr int kSliceTwo = 80 * 1024;
constexpr int kSliceOne = 176 * 1024;
constexpr int kMaxCluster = 8;
constexpr float kSpan = 32.f;                // of z in the bins: e^-32 of the weight is past them
constexpr float kFloatMax = 3.402823466e+38f;
constexpr uint32_t kLowest = 0x00800000u;    // order() of -FLT_MAX
constexpr int kAnyIndex = 0x7fffffff;

// Bit patterns in the order of the floats they hold (both zeros the same).
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unorder(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Larger of two packed pairs; of a number and a NaN the number.
template <int DT> __device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (DT == DT_BF16)
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int DT> constexpr uint32_t kMinusInfPair = DT == DT_BF16 ? 0xFF80FF80u : 0xFC00FC00u;

// One row's slice in a CTA: chunks of 16 bytes, aligned in memory, so the first and
// the last chunk of a row may be partly outside it (filled with -inf).
template <int DT, bool HELD> struct Slice {
  static constexpr int VE = DT == DT_F32 ? 4 : 8;
  using T = typename Elem<DT>::T;
  const T* row;
  uint4* held;         // shared memory (HELD), else the slice is read from global each time
  int64_t first;       // index of the first element of chunk 0 (may be negative)
  int chunks, vocab;
  bool infinite;       // the row's maximum is +inf: such logits count as 0, others as -inf
                       // (and are held so)

  __device__ __forceinline__ int64_t index(int j) const { return first + (int64_t)j * VE; }
  __device__ __forceinline__ bool inside(int j) const {
    return index(j) >= 0 && index(j) + VE <= vocab;
  }
  __device__ __forceinline__ uint4 load(int j) const {
    const int64_t at = index(j);
    if (inside(j)) return *reinterpret_cast<const uint4*>(row + at);
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < VE; ++i)
      e[i] = at + i >= 0 && at + i < vocab ? row[at + i] : Elem<DT>::from_f(-INFINITY);
    return u;
  }
  __device__ __forceinline__ uint4 at(int j) const {
    if constexpr (HELD) return held[j];
    return load(j);
  }
  // the chunk as floats, NaN as -inf
  __device__ __forceinline__ void get(int j, float (&x)[VE]) const { floats(at(j), x); }
  __device__ __forceinline__ void floats(const uint4 u, float (&x)[VE]) const {
    const uint32_t r[4] = {u.x, u.y, u.z, u.w};
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = fmaxf(__uint_as_float(r[i]), -INFINITY);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<DT>(max_pair<DT>(r[i], kMinusInfPair<DT>));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
    if constexpr (!HELD)
      if (infinite) {
#pragma unroll
        for (int i = 0; i < VE; ++i) x[i] = x[i] == INFINITY ? 0.f : -INFINITY;
      }
  }
  // rewrites this thread's chunks for a row whose maximum is +inf
  __device__ __forceinline__ void to_infinite() {
    infinite = true;
    if constexpr (HELD)
      for (int j = threadIdx.x; j < chunks; j += kThreads) {
        float x[VE];
        get(j, x);
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < VE; ++i) x[i] = x[i] == INFINITY ? 0.f : -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (DT == DT_F32)
            u[i] = __float_as_uint(x[i]);
          else
            u[i] = pack2<DT>(x[2 * i], x[2 * i + 1]);
        }
        held[j] = make_uint4(u[0], u[1], u[2], u[3]);
      }
  }
  // the largest logit of a chunk (NaN and a row with infinities aside: it may be too large)
  __device__ __forceinline__ float highest(int j) const { return highest_of(at(j)); }
  __device__ __forceinline__ static float highest_of(const uint4 u) {
    if constexpr (DT == DT_F32) {
      return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                   fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    } else {
      const float2 f = unpack2<DT>(max_pair<DT>(max_pair<DT>(u.x, u.y), max_pair<DT>(u.z, u.w)));
      return fmaxf(f.x, f.y);
    }
  }
  // the largest logit of this thread's chunks
  __device__ __forceinline__ float largest() const {
    float mx = -INFINITY;
    if constexpr (DT == DT_F32) {
      for (int j = threadIdx.x; j < chunks; j += kThreads) {
        float x[VE];
        get(j, x);
        mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), mx);
      }
    } else {
      uint32_t best = kMinusInfPair<DT>;
      for (int j = threadIdx.x; j < chunks; j += kThreads) {
        const uint4 u = at(j);
        best = max_pair<DT>(max_pair<DT>(max_pair<DT>(u.x, u.y), max_pair<DT>(u.z, u.w)), best);
      }
      const float2 f = unpack2<DT>(best);
      mx = fmaxf(f.x, f.y);
    }
    return mx;
  }
};

// A threshold: what is above x, and of what equals it the indices up to `last`.
struct Cut {
  float x;
  int last;
  __device__ __forceinline__ bool keeps(float v, int at) const {
    return v > x || (v == x && at <= last);
  }
};

template <int BYTES> __device__ __forceinline__ void copy_async(void* to, const void* from) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}

// This CTA's slice of row r.
template <int DT, bool HELD>
__device__ __forceinline__ Slice<DT, HELD> slice_of(const SampleArgs& a, cg::cluster_group& cl, int r, uint4* held) {
  using S = Slice<DT, HELD>;
  S sl;
  sl.row = reinterpret_cast<const typename S::T*>(a.logits) + r * a.logits_stride;
  sl.held = held;
  sl.vocab = a.vocab;
  sl.infinite = false;
  const int mis = (int)(reinterpret_cast<uintptr_t>(sl.row) % 16 / sizeof(typename S::T));
  const int all = (int)(((int64_t)mis + a.vocab + S::VE - 1) / S::VE);
  const int nblocks = (int)cl.num_blocks(), share = (all + nblocks - 1) / nblocks;
  const int c0 = min(all, (int)cl.block_rank() * share);
  sl.chunks = min(share, all - c0);
  sl.first = (int64_t)c0 * S::VE - mis;
  return sl;
}

struct Shared {
  unsigned hist[kBins];
  unsigned long long warp_best[kWarps];
  double sums[kWarps][4];
  double scan[kWarps];
  unsigned count;
  // written by this CTA, read by the cluster
  double row_sums[4];
  unsigned ties;
  float part_weight;
  // written by each CTA of the cluster, in its place
  unsigned long long least_of[kMaxCluster];
  unsigned top_of[kMaxCluster], bound_of[kMaxCluster], count_of[kMaxCluster];
  // in CTA 0: the best token and the sum of each CTA of the cluster
  unsigned long long best_of[kMaxCluster];
  double sum_of[kMaxCluster];
  // written by one CTA for all
  double share;
  // broadcast inside the CTA
  unsigned long long out_best;
  double out_sums[4];
  double found_above;
  unsigned found_bin, found_count;
  int part_start[kMaxCluster + 1];     // of each CTA's candidates in a merged list
  float part_total[kMaxCluster];       // and their weight
  int tie_last;
};

__device__ __forceinline__ unsigned long long pack(uint32_t key, int64_t at) {
  return (unsigned long long)key << 32 | (uint32_t)~(uint32_t)at;
}

__device__ __forceinline__ unsigned long long warp_best(unsigned long long v) {
  const unsigned key = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32));
  const unsigned low = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32) == key ? (unsigned)v : 0u);
  return (unsigned long long)key << 32 | low;
}

// Largest of `v` over the CTA, valid in warp 0.
__device__ unsigned long long block_best(Shared& sh, unsigned long long v) {
  v = warp_best(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp_best[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) v = warp_best(threadIdx.x < kWarps ? sh.warp_best[threadIdx.x] : 0ull);
  return v;
}

// Sums of N values over the CTA into row_sums from `slot`, in a fixed order (no barrier
// after; thread 0 may use them).
template <int N> __device__ void block_sum(Shared& sh, const float (&x)[N], int slot = 0) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    double v = x[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sh.sums[warp][i] = v;
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double v = lane < kWarps ? sh.sums[lane][i] : 0.0;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) sh.row_sums[slot + i] = v;
    }
  }
}

// Adds up row_sums[i] of the cluster's CTAs, in a fixed order; a warp calls it.
__device__ __forceinline__ double all_sums(cg::cluster_group& cl, Shared& sh, int i) {
  const unsigned lane = threadIdx.x & 31;
  double s = lane < cl.num_blocks() ? cl.map_shared_rank(&sh, lane)->row_sums[i] : 0.0;
#pragma unroll
  for (int o = 1; o < kMaxCluster; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return __shfl_sync(0xffffffffu, s, 0);
}

// Sums of N values over the cluster, in every thread.
template <int N> __device__ void cluster_sum(cg::cluster_group& cl, Shared& sh, const float (&x)[N], double (&v)[N]) {
  cl.sync();   // the last read of row_sums is over
  block_sum(sh, x);
  cl.sync();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = all_sums(cl, sh, i);
}

// Exclusive prefix of `v` over the CTA's threads.
__device__ double block_before(Shared& sh, double v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();   // the last use of scan is over
  if (lane == 31) sh.scan[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const double mine = lane < kWarps ? sh.scan[lane] : 0.0;
    double s = mine;
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane < kWarps) sh.scan[lane] = s - mine;
  }
  __syncthreads();
  return sh.scan[warp] + (incl - v);
}

// The settings of one row and its largest logit.
struct RowState {
  float heat, inv_heat, to_log2, top, scale;   // T, 1/T, log2(e)/T, bins per logit
  float top_p, min_p;

  __device__ __forceinline__ float z(float x) const { return __fdiv_rn(x - top, heat); }
  __device__ __forceinline__ float weight(float x) const { return ex2((x - top) * to_log2); }
  // bins as the floats 2^23 + bin (the addition rounds to whole bins); monotone in x
  __device__ __forceinline__ float place(float x) const {
    return fminf((top - x) * scale, (float)(kBins - 1)) + 8388608.f;
  }
  // 512 bins of the search by counting
  __device__ __forceinline__ int coarse(float x) const {
    return x == top ? 0 : (int)fminf((top - x) * scale * 0.5f, (float)(kThreads - 1));
  }
};

__device__ __forceinline__ RowState row_state(float heat, float top_p, float min_p) {
  RowState row;
  // its reciprocal stays finite and, if subnormal, above 0: an infinite one counts as the largest
  row.heat = heat > 0.f ? fminf(fmaxf(heat, 1e-30f), kFloatMax) : 1.f;
  row.inv_heat = 1.f / row.heat;
  row.to_log2 = row.inv_heat * kLog2e;
  row.scale = (float)kBins / kSpan * row.inv_heat;
  row.top = 0.f;
  row.top_p = top_p;
  row.min_p = min_p;
  return row;
}

// Settings that leave the largest logit's first token alone.
__host__ __device__ inline bool takes_largest(float heat, int top_k, float top_p, float min_p) {
  return !(heat > 0.f) || top_k == 1 || !(top_p > 0.f) || !(min_p <= 1.f);
}

// Descending bitonic sort of the n <= kList values of `v` (shared memory) by the first
// warps of the CTA, four values a thread in registers: steps of 1 and 2 inside a
// thread, up to 64 by shuffles, above through shared memory. Past n there are zeros up
// to a whole number of threads. The whole CTA calls it; on return thread i holds the
// values 4 i to 4 i + 3 (0 past the warps that sorted).
__device__ void sort_down(unsigned long long* v, int n, unsigned long long (&x)[4]) {
  int n2 = 128;   // a warp
  while (n2 < n) n2 <<= 1;
  const int tid = threadIdx.x, threads = n2 / 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = 0;
  __syncthreads();
  if (tid >= threads) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (4 * tid + i < n) x[i] = v[4 * tid + i];
  auto swap = [](unsigned long long& p, unsigned long long& q, bool down) {
    const bool change = (p < q) == down;
    const unsigned long long u = change ? q : p, w = change ? p : q;
    p = u;
    q = w;
  };
  swap(x[0], x[1], true);
  swap(x[2], x[3], false);
  for (int size = 4; size <= n2; size <<= 1) {
    const bool down = (4 * tid & size) == 0;
    for (int step = size >> 1; step >= 128; step >>= 1) {
      if (threads > 32) named_bar_sync(1, threads);   // the last round's reads are over
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * tid + i] = x[i];
      named_bar_sync(1, threads);
      const bool keep_large = ((4 * tid & step) == 0) == down;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned long long y = v[(4 * tid + i) ^ step];
        x[i] = (x[i] > y) == keep_large ? x[i] : y;
      }
    }
    for (int step = min(size >> 1, 64); step >= 4; step >>= 1) {
      const bool keep_large = ((4 * tid & step) == 0) == down;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, x[i], step >> 2);
        x[i] = (x[i] > y) == keep_large ? x[i] : y;
      }
    }
    swap(x[0], x[2], down);
    swap(x[1], x[3], down);
    swap(x[0], x[1], down);
    swap(x[2], x[3], down);
  }
}

// Sets part_start to where each CTA's candidates start in a list of all of them, from
// lane r's number of CTA r's; returns the number of all. Every warp calls it; the other
// warps may use part_start after a barrier.
__device__ int place_parts(Shared& sh, int c) {
  const int lane = threadIdx.x & 31;
  int upto = c;
#pragma unroll
  for (int o = 1; o < kMaxCluster; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (threadIdx.x < kMaxCluster) sh.part_start[lane + 1] = upto;   // past the last CTA: the end
  if (threadIdx.x == 0) sh.part_start[0] = 0;
  return __shfl_sync(0xffffffffu, upto, kMaxCluster - 1);
}

// Once a CTA's candidates are gathered: tells the others their number and waits for the
// cluster; then as above.
__device__ int exchange_parts(cg::cluster_group& cl, Shared& sh) {
  const int lane = threadIdx.x & 31, nblocks = (int)cl.num_blocks();
  __syncthreads();
  if ((int)threadIdx.x < nblocks) cl.map_shared_rank(&sh, threadIdx.x)->count_of[cl.block_rank()] = sh.count;
  cl.sync();
  return place_parts(sh, lane < nblocks ? (int)sh.count_of[lane] : 0);
}

// The largest number of candidates a CTA has.
__device__ __forceinline__ int largest_part(Shared& sh, int nblocks) {
  int most = 0;
  for (int q = 0; q < nblocks; ++q) most = max(most, (int)sh.count_of[q]);
  return most;
}

// Sorts the cluster's candidates: afterwards every CTA has all of them, each CTA's part
// (from part_start) sorted (descending, ties by index ascending) with the running weight
// of the part before each. All CTAs call it, after part_start was set.
__device__ void merge_lists(cg::cluster_group& cl, Shared& sh, const RowState& row, unsigned long long* list,
                            float* ahead) {
  const int tid = threadIdx.x, me = (int)cl.block_rank(), nblocks = (int)cl.num_blocks();
  __syncthreads();
  const int start = sh.part_start[me], own = sh.part_start[me + 1] - start;
  unsigned long long v[4];
  if (own <= kFew / 2) {   // four threads a candidate count the larger ones
    const int i = tid >> 2;
    v[0] = i < own ? list[i] : 0;
    int place = 0;
    if (i < own)
      for (int j = tid & 3; j < own; j += 4) place += list[j] > v[0];
    place += __shfl_xor_sync(0xffffffffu, place, 1);
    place += __shfl_xor_sync(0xffffffffu, place, 2);
    __syncthreads();
    if (i < own && (tid & 3) == 0) list[start + place] = v[0];
  } else {
    sort_down(list, own, v);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * tid + i < own) list[start + 4 * tid + i] = v[i];
  }
  __syncthreads();
  const int each = (own + kThreads - 1) / kThreads;   // at most 4
  float w[4];
  double mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = each * tid + i;
    w[i] = i < each && at < own ? row.weight(unorder((uint32_t)(list[start + at] >> 32))) : 0.f;
    mine += w[i];
  }
  double run = block_before(sh, mine);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = each * tid + i;
    if (i < each && at < own) ahead[start + at] = (float)run;
    run += w[i];
  }
  if (tid == kThreads - 1) sh.part_weight = (float)run;
  cl.sync();
  const int all = sh.part_start[nblocks];
  for (int i = tid; i < all; i += kThreads) {
    int c = 0;
#pragma unroll
    for (int q = 1; q < kMaxCluster; ++q) c += i >= sh.part_start[q];
    const unsigned long long key = cl.map_shared_rank(list, c)[i];
    const float f = cl.map_shared_rank(ahead, c)[i];
    list[i] = key;   // its own ones with what they are
    ahead[i] = f;
  }
  if (tid < nblocks) sh.part_total[tid] = cl.map_shared_rank(&sh, tid)->part_weight;
  __syncthreads();
}

// Calls each(place in this CTA's part, candidate, number of larger ones, their weight) for
// this CTA's candidates after merge_lists(), each by one thread: as many lanes as the
// cluster has CTAs share a candidate and search a part each.
template <typename F>
__device__ __forceinline__ void for_places(Shared& sh, const unsigned long long* list, const float* ahead, int me,
                                           int nblocks, const F& each) {
  const int start = sh.part_start[me], own = sh.part_start[me + 1] - start;
  const int c = threadIdx.x & (nblocks - 1);   // a power of two
  const int s0 = sh.part_start[c], n = sh.part_start[c + 1] - s0;
  const int per = kThreads / nblocks;
  for (int i0 = 0; i0 < own; i0 += per) {
    const int i = i0 + (int)threadIdx.x / nblocks;
    const unsigned long long v = i < own ? list[start + i] : ~0ull;
    int lo = 0;   // known to be larger
    for (int step = n > 0 ? 1 << (31 - __clz(n)) : 0; step > 0; step >>= 1) {
      const int to = lo + step;
      lo = to <= n && list[s0 + min(to, n) - 1] > v ? to : lo;
    }
    float before = n == 0 ? 0.f : lo < n ? ahead[s0 + lo] : sh.part_total[c];
    for (int o = 1; o < nblocks; o <<= 1) {
      lo += __shfl_xor_sync(0xffffffffu, lo, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (c == 0 && i < own) each(i, v, lo, before);
  }
}

__device__ __forceinline__ void gather(Shared& sh, unsigned long long* list, float x, int64_t at) {
  const unsigned i = atomicAdd(&sh.count, 1u);
  if (i < kList) list[i] = pack(order(x), at);
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// Adds up bin threadIdx.x of the cluster's CTAs and clears it.
__device__ unsigned gather_bin(cg::cluster_group& cl, Shared& sh) {
  cl.sync();
  unsigned c = 0;
#pragma unroll
  for (unsigned r = 0; r < kMaxCluster; ++r)
    if (r < cl.num_blocks()) c += cl.map_shared_rank(&sh, r)->hist[threadIdx.x];
  cl.sync();
  sh.hist[threadIdx.x] = 0;
  return c;
}

// Search by counting for the value where the ordered logits within `within` reach
// `target` (a count, or a weight). On return the crossing value is `key` with `count`
// logits equal to it and `above` of the target used up by larger ones; or, when not
// `single`, `key` is a lower bound, and what reaches it is just what is needed.
//
// Logits are counted in bins, first linear in x, then over the bit patterns of the bin that the
// target falls into, until a bin is one value. Until then counts only say about where a weight
// is reached: a bin is off by as much as the weights in it differ (30 of 8000 tokens, where
// it is half a power of two wide, at zero). So the weights above and in three bins there are
// added up, and the three are moved on until the target lies in them.
struct Found {
  uint32_t key;
  unsigned count;
  double above;
  bool single;
};

template <int DT, bool HELD, bool WEIGHT>
__device__ Found search(cg::cluster_group& cl, Shared& sh, const Slice<DT, HELD>& sl, const RowState& row,
                        double target, const Cut& within) {
  constexpr int VE = Slice<DT, HELD>::VE;
  const int tid = threadIdx.x;
  const uint32_t least = order(fmaxf(within.x, -kFloatMax));
  uint32_t lo = least, hi = order(row.top);
  double above = 0;
  unsigned count = 0xffffffffu;   // not known
  bool linear = true;
  int shift = 0;
  // calls each(logit, its bin) for those in the range
  auto for_bins = [&](auto each) {
    for (int j = tid; j < sl.chunks; j += kThreads) {
      float x[VE];
      sl.get(j, x);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const uint32_t k = order(x[i]);
        if (k >= lo && k <= hi) each(x[i], linear ? row.coarse(x[i]) : (int)((hi - k) >> shift));
      }
    }
  };
  while (true) {
    if (!linear) {
      if (!WEIGHT && above + (double)count <= target) return {lo, count, above, false};
      if (count <= 1) return {lo, count, above, false};   // 0: rounding let the target end with what is above
      if (lo >= hi && count != 0xffffffffu) return {lo, count, above, true};
      const int bits = 32 - __clz((hi - lo) | 1);   // keys less one
      shift = bits > kKeyBits ? bits - kKeyBits : 0;
    }
    for_bins([&](float, int b) { atomicAdd(&sh.hist[b], 1u); });
    const unsigned c = gather_bin(cl, sh);
    const uint32_t span = (1u << shift) - 1, off = (uint32_t)tid << shift;
    double mass = (double)c;
    if (WEIGHT && c != 0) {   // as its middle
      mass *= linear ? (double)ex2(-((float)tid + (tid == 0 ? 0.f : 0.5f)) * (kSpan / (float)kThreads * kLog2e))
                     : (double)row.weight(unorder(hi - off - min(span / 2, (hi - off - lo) / 2)));
    }
    const double before = block_before(sh, mass) + above;
    __syncthreads();
    if (tid == 0) sh.found_bin = 0xffffffffu;
    __syncthreads();
    if (c != 0 && before + mass >= target) atomicMin(&sh.found_bin, (unsigned)tid);
    __syncthreads();
    if (sh.found_bin == 0xffffffffu) {   // rounding left the target just past the last value: take that one
      __syncthreads();
      if (tid == 0) sh.found_bin = 0;
      __syncthreads();
      if (c != 0) atomicMax(&sh.found_bin, (unsigned)tid);
      __syncthreads();
    }
    int bin = (int)sh.found_bin;
    if (tid == bin) sh.found_above = before;
    if (WEIGHT && (linear || shift > 0)) {
      int moved = 0;
      while (true) {
        bin = min(max(bin, 1), kThreads - 2);
        float s[4] = {0.f, 0.f, 0.f, 0.f};   // above, and in the three
        for_bins([&](float x, int b) {
          if (b > bin + 1) return;
          const float w = row.weight(x);
          s[0] += b < bin - 1 ? w : 0.f;
          s[1] += b == bin - 1 ? w : 0.f;
          s[2] += b == bin ? w : 0.f;
          s[3] += b == bin + 1 ? w : 0.f;
        });
        double v[4];
        cluster_sum(cl, sh, s, v);
        // a step that would turn back has met the crossing
        if (above + v[0] >= target && bin > 1 && moved <= 0) {
          bin -= 3;
          moved = -1;
          continue;
        }
        if (above + v[0] + v[1] + v[2] + v[3] < target && bin < kThreads - 2 && moved >= 0) {
          bin += 3;
          moved = 1;
          continue;
        }
        above += v[0];
        --bin;
        if (above + v[1] < target) {
          above += v[1];
          ++bin;
          if (above + v[2] < target) {
            above += v[2];
            ++bin;
          }
        }
        break;
      }
      if (tid == bin) sh.found_above = above;
    }
    if (tid == bin) sh.found_count = c;
    __syncthreads();
    above = sh.found_above;
    count = sh.found_count;
    if (linear) {
      // the keys of the bin: coarse() falls as the key grows
      linear = false;
      if (bin < kThreads - 1) {   // smallest key whose bin is <= bin
        uint32_t a = kLowest, b = hi;
        while (a < b) {
          const uint32_t mid = a + (b - a) / 2;
          if (row.coarse(unorder(mid)) <= bin) b = mid; else a = mid + 1;
        }
        lo = max(a, least);
      }
      if (bin > 0) {           // largest key whose bin is >= bin
        uint32_t a = lo, b = hi;
        while (a < b) {
          const uint32_t mid = a + (b - a + 1) / 2;
          if (row.coarse(unorder(mid)) >= bin) a = mid; else b = mid - 1;
        }
        hi = a;
      }
    } else {
      hi -= (uint32_t)bin << shift;
      if (hi - lo > span) lo = hi - span;
    }
    __syncthreads();
  }
}

// Index of the `need`-th logit (from 1) equal to `value`, in index order.
template <int DT, bool HELD>
__device__ int tie_index(cg::cluster_group& cl, Shared& sh, const Slice<DT, HELD>& sl, float value, unsigned need) {
  constexpr int VE = Slice<DT, HELD>::VE;
  const int share = (sl.chunks + kThreads - 1) / kThreads;   // chunks a thread, consecutive
  const int j0 = min(sl.chunks, (int)threadIdx.x * share), j1 = min(sl.chunks, j0 + share);
  unsigned mine = 0;
  for (int j = j0; j < j1; ++j) {
    float x[VE];
    sl.get(j, x);
#pragma unroll
    for (int i = 0; i < VE; ++i) mine += x[i] == value;
  }
  const unsigned before = (unsigned)block_before(sh, (double)mine);
  if (threadIdx.x == kThreads - 1) {
    sh.ties = before + mine;
    sh.tie_last = -1;
  }
  cl.sync();
  unsigned ahead = 0;
  for (unsigned r = 0; r < cl.block_rank(); ++r) ahead += cl.map_shared_rank(&sh, r)->ties;
  const unsigned from = ahead + before;
  if (from < need && need <= from + mine) {
    unsigned seen = from;
    for (int j = j0; j < j1; ++j) {
      float x[VE];
      sl.get(j, x);
      for (int i = 0; i < VE; ++i)
        if (x[i] == value && ++seen == need) {
          const int at = (int)(sl.index(j) + i);
          for (unsigned r = 0; r < cl.num_blocks(); ++r) cl.map_shared_rank(&sh, r)->tie_last = at;
        }
    }
  }
  cl.sync();
  return sh.tie_last;
}

__device__ __forceinline__ float race_score(float z, float e) {
  return e > 0.f ? z - logf(e) : -3.402823466e+38f;   // noise has to be positive
}

// The smallest logit whose weight reaches min_p in (0, 1]; every lane of a warp calls it.
__device__ float min_p_logit(const RowState& row) {
  const int lane = threadIdx.x & 31;
  uint32_t lo = kLowest, hi = order(row.top);   // hi reaches it: its weight is 1
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 32 + 1;
    const uint64_t mine = (uint64_t)lo + (uint64_t)lane * step;
    const bool reaches = mine >= hi || expf(row.z(unorder((uint32_t)mine))) >= row.min_p;
    const int at = __ffs(__ballot_sync(0xffffffffu, reaches)) - 1;   // first lane that reaches it, -1: none
    const uint32_t base = lo;
    if (at != 0) lo = base + (uint32_t)(at < 0 ? 31 : at - 1) * step + 1;
    if (at >= 0) hi = min(hi, base + (uint32_t)at * step);
  }
  return unorder(hi);
}

// Top-p over the whole row: cut after the shortest prefix with p of the weight.
// Returns false (everywhere) when the crossing bin does not fit the list or lies below the others.
template <int DT, bool HELD>
__device__ bool nucleus(cg::cluster_group& cl, Shared& sh, const Slice<DT, HELD>& sl, RowState row,
                        unsigned long long* list, float* ahead, double& whole, Cut& cut) {
  constexpr int VE = Slice<DT, HELD>::VE;
  const int tid = threadIdx.x;
  // Tokens with less than (1 - p) / vocab of the largest one's weight do not reach 1 - p of
  // all weight together, so the prefix ends above them: the bins span the rest.
  const float span = fminf(kSpan, logf((float)sl.vocab) - logf(fmaxf(1.f - row.top_p, 1e-9f)) + 0.1f);
  row.scale *= kSpan / span;
  float s[1] = {0.f};
#pragma unroll 2
  for (int j = tid; j < sl.chunks; j += kThreads) {
    float x[VE];
    sl.get(j, x);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      s[0] += row.weight(x[i]);
      const int b = __float_as_int(row.place(x[i])) & (kBins - 1);
      if (b < kBins - 1) atomicAdd(&sh.hist[b], 1u);
    }
  }
  block_sum(sh, s);
  cl.sync();
  unsigned c0 = 0, c1 = 0;
#pragma unroll
  for (unsigned r = 0; r < kMaxCluster; ++r)
    if (r < cl.num_blocks()) {
      const uint2 u = reinterpret_cast<const uint2*>(cl.map_shared_rank(&sh, r)->hist)[tid];
      c0 += u.x;
      c1 += u.y;
    }
  whole = all_sums(cl, sh, 0);
  if (tid == 0) sh.found_bin = kBins - 3;
  // A bin weighs about its count times its middle's weight. The crossing is looked for in
  // two bins, the one where the estimates cross and the neighbour on the nearer side: the
  // largest tokens are few, and where they lie in their bins is not averaged out.
  const float per_bin = row.to_log2 / row.scale;
  const double m0 = (double)c0 * ex2(-(tid == 0 ? 0.25f : 2.f * tid) * per_bin);
  const double m1 = (double)c1 * ex2(-(2.f * tid + 1.f) * per_bin);
  const double start = block_before(sh, m0 + m1);
  const double target = (double)row.top_p * whole;
  if (start + m0 + m1 >= target) {
    const bool second = start + m0 < target;
    const bool low_half = target - start - (second ? m0 : 0.0) < 0.5 * (second ? m1 : m0);
    const int lower = 2 * tid + (second ? 1 : 0) - (low_half ? 1 : 0);
    atomicMin(&sh.found_bin, (unsigned)min(max(lower, 0), kBins - 3));
  }
  __syncthreads();
  int bin = (int)sh.found_bin, moved = 0;   // the lower one of the two
  for (int tries = 0; tries < 16; ++tries) {
    // how many of the bins' logits each CTA has
    int mine = 0;
    if ((tid & 31) < (int)cl.num_blocks()) {
      const unsigned* hist = cl.map_shared_rank(&sh, tid & 31)->hist;
      mine = (int)(hist[bin] + hist[bin + 1]);
    }
    const int n = place_parts(sh, mine);
    if (n > kList) return false;
    // the weight above the bins, and the bins' logits
    const float at_bin = 8388608.f + (float)bin;
    float a[1] = {0.f};
#pragma unroll 2
    for (int j = tid; j < sl.chunks; j += kThreads) {
      float x[VE];
      sl.get(j, x);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float p = row.place(x[i]);
        if (p < at_bin) a[0] += row.weight(x[i]);
        if (p == at_bin || p == at_bin + 1.f) gather(sh, list, x[i], sl.index(j) + i);
      }
    }
    const int slot = 1 + (tries & 1);   // the other one may still be read
    block_sum(sh, a, slot);
    merge_lists(cl, sh, row, list, ahead);
    const double above = all_sums(cl, sh, slot);
    // the last one that the prefix has to take: the smallest with less than the target before it
    unsigned long long least = 0;   // inverted, so that the smallest is the best
    for_places(sh, list, ahead, (int)cl.block_rank(), (int)cl.num_blocks(), [&](int, unsigned long long v, int, float before) {
      if (above + before < target) least = max(least, ~v);
    });
    least = __shfl_sync(0xffffffffu, block_best(sh, least), 0);
    if (tid < (int)cl.num_blocks()) cl.map_shared_rank(&sh, tid)->least_of[cl.block_rank()] = least;
    double total = above;
    for (unsigned r = 0; r < cl.num_blocks(); ++r) total += sh.part_total[r];
    cl.sync();
    least = warp_best((tid & 31) < (int)cl.num_blocks() ? sh.least_of[tid & 31] : 0ull);
    if (tid == 0) sh.count = 0;
    __syncthreads();
    // a step that would turn back has met the crossing
    if (above >= target && bin > 0 && moved <= 0) {
      moved = -1;
      bin = max(bin - 2, 0);
    } else if (total < target && bin < kBins - 3 && moved >= 0) {
      moved = 1;
      bin = min(bin + 2, kBins - 3);
    } else if (total < target && bin >= kBins - 3) {
      return false;   // the prefix ends below the bins (millions of tokens past 32 nats, or rounding)
    } else {
      if (least == 0) {   // nothing of the bin is needed
        cut.x = row.top - ((float)bin - 0.5f) / row.scale;
        cut.last = kAnyIndex;
      } else {
        cut.x = unorder((uint32_t)(~least >> 32));
        cut.last = (int)(uint32_t)least;
      }
      return true;
    }
  }
  return false;
}

// A row's noise beside its slice of logits.
template <int DT, bool HELD> struct Noise {
  static constexpr int VE = Slice<DT, HELD>::VE;
  const float* noise;
  const int4* words;
  int whole0, whole1;   // chunks whose noise is whole 16-byte words: all but a row's first and last, or none

  __device__ __forceinline__ Noise(const Slice<DT, HELD>& sl, const float* noise) : noise(noise) {
    const bool aligned = reinterpret_cast<uintptr_t>(noise + sl.first) % 16 == 0;
    whole0 = sl.chunks > 0 && !sl.inside(0) ? 1 : 0;
    whole1 = !aligned ? 0 : sl.chunks > 0 && !sl.inside(sl.chunks - 1) ? sl.chunks - 1 : sl.chunks;
    words = reinterpret_cast<const int4*>(noise + sl.first);
  }
  // bit patterns of chunk j's, left as they are outside the row
  __device__ __forceinline__ void fetch(const Slice<DT, HELD>& sl, int j, int (&to)[VE]) const {
    if (j >= whole0 && j < whole1) {
#pragma unroll
      for (int i = 0; i < VE; i += 4) {
        const int4 f = __ldcs(words + j * (VE / 4) + i / 4);
        to[i] = f.x, to[i + 1] = f.y, to[i + 2] = f.z, to[i + 3] = f.w;
      }
    } else {
      const int64_t at = sl.index(j);
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (at + i >= 0 && at + i < sl.vocab) to[i] = __float_as_int(noise[at + i]);
    }
  }
};

// The race's rough score: t less the logarithm of noise with this bit pattern. 2^23 + bits / 2^8
// is exact as a float: 2^15 (k + m) and a constant.
__device__ __forceinline__ float rough_score(float t, int bits) {
  return fmaf(__int_as_float(0x4B000000 | bits >> 8), -0x1p-15f, t);
}
constexpr float kReach = 0.0861f + 1e-3f;   // the log's error, and the rounding of scores to about 500

// The best token by exact scores, given every thread's best and second best rough score of
// its chunks, the best one's chunk, and the smallest noise pattern it saw.
template <int DT, bool HELD>
__device__ __forceinline__ unsigned long long race_end(Shared& sh, const Slice<DT, HELD>& sl, const RowState& row,
                                                       const Cut cut, const float* noise, float best,
                                                       float second, int best_j, int least, bool any) {
  constexpr int VE = Slice<DT, HELD>::VE;
  const int tid = threadIdx.x;
  const unsigned high = __reduce_max_sync(0xffffffffu, order(best));
  __syncthreads();
  if ((tid & 31) == 0) sh.warp_best[tid >> 5] = high;
  // noise that is no positive normal number has no such logarithm: all is scored exactly
  bool odd = __syncthreads_or(least < 0x00800000);
  any = __syncthreads_or(any);
  const unsigned cta =
      __reduce_max_sync(0xffffffffu, (unsigned)sh.warp_best[tid & (kWarps - 1)]);
  const float bar = unorder(cta) - kReach;
  odd |= any && !(bar > -INFINITY);
  unsigned long long best_key = 0;
  if (odd || best >= bar) {
    const bool every = odd || second >= bar;
    for (int j = every ? tid : best_j; j < sl.chunks; j += every ? kThreads : 0x40000000) {
      float x[VE], n[VE];
      sl.get(j, x);
      const int at = (int)sl.first + j * VE;
#pragma unroll
      for (int i = 0; i < VE; ++i) n[i] = at + i >= 0 && at + i < sl.vocab ? noise[at + i] : INFINITY;
#pragma unroll 1
      for (int i = 0; i < VE; ++i) {
        float mine = x[0], its = n[0];
#pragma unroll
        for (int q = 1; q < VE; ++q) {
          mine = i == q ? x[q] : mine;
          its = i == q ? n[q] : its;
        }
        if (!cut.keeps(mine, at + i) ||
            (!odd && rough_score((mine - row.top) * row.to_log2, __float_as_int(its)) < bar))
          continue;
        const float z = row.z(mine);
        if (z > -INFINITY) best_key = max(best_key, pack(order(race_score(z, its)), at + i));
      }
    }
  }
  return best_key;
}
// The race over a CTA's tokens that the cut keeps: its best
// pack(order(score), index), thread by thread. With sum_here the weights of all tokens
// are added to `sum`.
//
// A thread's noise is loaded 16 values ahead of their use. Scores are first taken
// roughly, in powers of two: for e = 2^k (1 + m) the exponent and mantissa bits read as one
// number are k + m = log2 e - [0, 0.0861], three integer and float operations in place of
// the special-function unit's, which the weights' exponentials keep busy. A thread keeps
// its best chunk of them; then only the chunks within reach of the CTA's best are scored
// exactly.
template <int DT, bool HELD>
__device__ __forceinline__ unsigned long long race(Shared& sh, const Slice<DT, HELD>& sl, const RowState& row,
                                                   const Cut cut, const float* noise, bool sum_here, float& sum) {
  constexpr int VE = Slice<DT, HELD>::VE, DEPTH = 16 / VE;
  const int tid = threadIdx.x;
  const Noise<DT, HELD> from(sl, noise);
  int e[DEPTH][VE];   // bit patterns
  auto fetch = [&](int j, int (&to)[VE]) {
#pragma unroll
    for (int i = 0; i < VE; ++i) to[i] = 0x7F800000;
    if (j >= sl.chunks || !(sl.highest(j) >= cut.x)) return;
    from.fetch(sl, j, to);
  };
#pragma unroll
  for (int u = 0; u < DEPTH; ++u) fetch(tid + u * kThreads, e[u]);
  float best = -INFINITY, second = -INFINITY;   // of the thread's chunks
  int best_j = 0, least = 0x7F800000;
  bool any = false;
  for (int jw = tid; jw < sl.chunks; jw += DEPTH * kThreads) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) {
      const int j = jw + u * kThreads;
      if (j < sl.chunks) {
        float x[VE], near = -INFINITY;
        sl.get(j, x);
        const int at = (int)sl.first + j * VE;
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float t = (x[i] - row.top) * row.to_log2;
          if (sum_here) sum += ex2(t);
          least = min(least, e[u][i]);
          const float score = rough_score(t, e[u][i]);
          if (cut.keeps(x[i], at + i)) {
            near = fmaxf(near, score);
            any = true;
          }
        }
        if (near > best) {
          second = best;
          best = near;
          best_j = j;
        } else {
          second = fmaxf(second, near);
        }
        fetch(j + DEPTH * kThreads, e[u]);
      }
    }
  }
  return race_end(sh, sl, row, cut, noise, best, second, best_j, least, any);
}

// Hands a CTA's best token and its part of the sum (thread 0's) to CTA 0. True for the
// other CTAs, which have arrived and may leave: nothing of theirs is read after this.
__device__ __forceinline__ bool leave(cg::cluster_group& cl, Shared& sh, unsigned long long best, double part) {
  if (threadIdx.x == 0) {
    Shared* to = cl.map_shared_rank(&sh, 0);
    to->best_of[cl.block_rank()] = best;
    to->sum_of[cl.block_rank()] = part;
  }
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  if (cl.block_rank() != 0) return true;
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  return false;
}

// CTA 0, after leave(): the row's token, and its log-probability.
template <int DT, bool HELD>
__device__ __forceinline__ void finish(const SampleArgs& a, Shared& sh, const Slice<DT, HELD>& sl,
                                       const RowState& row, int r, int nblocks) {
  __syncthreads();
  if (threadIdx.x < 32) {
    const unsigned long long v = warp_best(threadIdx.x < nblocks ? sh.best_of[threadIdx.x] : 0ull);
    double sum = threadIdx.x < nblocks ? sh.sum_of[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) {
      const int token = (int)~(uint32_t)v;
      a.tokens[r] = token;
      if (a.logprobs != nullptr) {
        const float x = sl.infinite ? 0.f : Elem<DT>::to_f(sl.row[token]);
        a.logprobs[r] = (float)((double)row.z(x) - log(sum));
      }
    }
  }
}

// A row that nothing filters, or of which the largest is taken (GREEDY): it is read once and
// not held. A thread takes its scores and weights relative to a logit of its own, moved when
// one passes it by 8 powers of two; the row's maximum is exchanged when all is read. Chunks
// on their way are in shared memory: loads to registers
// would have to pass what the other uses of shared memory leave of the L1 (200 rows of 151936
// bf16 54.8 us so, 44.8 us now).
constexpr int kStages = 4;
template <int DT> constexpr int kStreamBytes = kStages * kThreads * 16 * (1 + Slice<DT, false>::VE / 4);

template <int DT, bool GREEDY>
__device__ __forceinline__ void stream_row(const SampleArgs& a, cg::cluster_group& cl, Shared& sh,
                                           Slice<DT, false> sl, RowState row, const float* noise, int r,
                                           unsigned char* ring) {
  constexpr int VE = Slice<DT, false>::VE, PARTS = 1 + VE / 4;
  const int tid = threadIdx.x, rank = (int)cl.block_rank(), nblocks = (int)cl.num_blocks();
  const bool want_sum = a.logprobs != nullptr;
  const int lane = tid & 31;
  const bool aligned = reinterpret_cast<uintptr_t>(noise + sl.first) % 16 == 0;
  // a warp's stage: 32 chunks of logits, then their noise, in pieces of 16 bytes; with two
  // pieces a chunk every other eight are swapped in pairs, for threads' reads to differ in banks
  uint4* const stages = reinterpret_cast<uint4*>(ring) + (tid - lane) * PARTS;
  auto piece = [](int c) { return 32 + (PARTS == 3 ? c ^ (c >> 3 & 1) : c); };
  // chunks j0 to j0 + 31, whose noise the lanes copy in its order in memory
  auto issue = [&](int j0, int stage) {
    if (j0 < sl.chunks) {
      uint4* const to = stages + stage * PARTS * kThreads;
      const int j = j0 + lane;
      const bool whole = !GREEDY && j0 + 31 < sl.chunks && sl.inside(j0) && sl.inside(j0 + 31);
      if (whole || (j < sl.chunks && sl.inside(j)))
        copy_async<16>(to + lane, sl.row + sl.index(j));
      else if (j < sl.chunks)
        to[lane] = sl.load(j);
      if constexpr (!GREEDY) {
        if (whole && aligned) {
          const float* e = noise + sl.index(j0);
#pragma unroll
          for (int c = lane; c < 32 * (PARTS - 1); c += 32) copy_async<16>(to + piece(c), e + 4 * c);
        } else if (j < sl.chunks) {
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const int64_t at = sl.index(j) + i;
            float* const one = reinterpret_cast<float*>(to + piece(lane * (PARTS - 1) + i / 4)) + i % 4;
            if (at >= 0 && at < sl.vocab)
              copy_async<4>(one, noise + at);
            else
              *one = INFINITY;
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(tid - lane + i * kThreads, i);
  const float slack = fminf(8.f / row.to_log2, kFloatMax);   // finite: added to a reference of -inf
  float ref = -INFINITY, base = 0.f, most = -INFINITY, sum = 0.f;   // base: ref, or 0 for -inf
  float best = -INFINITY, second = -INFINITY;
  int best_j = 0, least = 0x7F800000, stage = 0;
  for (int j0 = tid - lane; j0 < sl.chunks; j0 += kThreads) {
    if constexpr (!GREEDY) __syncwarp();   // the last round's reads are over
    issue(j0 + (kStages - 1) * kThreads, (stage + kStages - 1) % kStages);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    if constexpr (!GREEDY) __syncwarp();
    const uint4* const from = stages + stage * PARTS * kThreads;
    stage = (stage + 1) % kStages;
    const int j = j0 + lane;
    if (j >= sl.chunks) continue;
    const uint4 u = from[lane];
    const float high = Slice<DT, false>::highest_of(u);
    if (GREEDY && high > most) best_j = j;
    most = fmaxf(most, high);
    if (high > ref + slack) {
      const float by = (ref - high) * row.to_log2;
      sum *= ex2(by);
      best += by;
      second += by;
      ref = base = high;
    }
    if (GREEDY && !want_sum) continue;
    float x[VE], near = -INFINITY;
    sl.floats(u, x);
    int e[VE];
    if constexpr (!GREEDY) {
#pragma unroll
      for (int p = 1; p < PARTS; ++p) {
        const uint4 w = from[piece(lane * (PARTS - 1) + p - 1)];
        e[4 * p - 4] = (int)w.x, e[4 * p - 3] = (int)w.y, e[4 * p - 2] = (int)w.z, e[4 * p - 1] = (int)w.w;
      }
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float t = (x[i] - base) * row.to_log2;
      if (want_sum) sum += ex2(t);
      if constexpr (!GREEDY) {
        least = min(least, e[i]);
        near = fmaxf(near, rough_score(t, e[i]));
      }
    }
    if constexpr (!GREEDY) {
      if (near > best) {
        second = best;
        best = near;
        best_j = j;
      } else {
        second = fmaxf(second, near);
      }
    }
  }

  // the row's maximum
  {
    const unsigned high = __reduce_max_sync(0xffffffffu, order(most));
    if ((tid & 31) == 0) sh.warp_best[tid >> 5] = high;
    __syncthreads();
    const unsigned of_cta = __reduce_max_sync(0xffffffffu, (unsigned)sh.warp_best[tid & (kWarps - 1)]);
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (tid < nblocks) cl.map_shared_rank(&sh, tid)->top_of[rank] = of_cta;
  }
  cl.sync();
  unsigned top = 0;
  for (int q = 0; q < nblocks; ++q) top = max(top, sh.top_of[q]);
  row.top = unorder(top);
  if (row.top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = -1;
      if (want_sum) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  unsigned long long key = 0;
  float s[1] = {sum * ex2((ref - row.top) * row.to_log2)};
  if (row.top == INFINITY) {
    sl.infinite = true;   // such logits count as 0, others as -inf
    row.top = 0.f;
    s[0] = 0.f;
    for (int j = tid; j < sl.chunks; j += kThreads) {
      float x[VE];
      sl.get(j, x);
#pragma unroll
      for (int i = 0; i < VE; ++i) s[0] += row.weight(x[i]);
    }
    if (!GREEDY) least = 0;   // all is scored exactly
  }
  if constexpr (GREEDY) {
    // the first of this thread's that equal the maximum are in its chunk best_j
    if (sl.chunks > tid) {
      float x[VE];
      sl.get(best_j, x);
      unsigned at = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (x[i] == row.top) at = min(at, (unsigned)(sl.index(best_j) + i));
      if (at != 0xffffffffu) key = pack(1u, at);
    }
  } else {
    const float by = (ref - row.top) * row.to_log2;
    key = race_end(sh, sl, row, Cut{-kFloatMax, kAnyIndex}, noise, best + by, second + by, best_j, least,
                   sl.chunks > 0);
  }
  key = block_best(sh, key);
  if (want_sum) block_sum(sh, s, 3);
  if (leave(cl, sh, key, want_sum ? sh.row_sums[3] : 0.0)) return;
  finish(a, sh, sl, row, r, nblocks);
}

// Rows whose settings are all known at launch to need stream_row().
template <int DT, bool GREEDY>
__global__ void __launch_bounds__(kThreads, 2) sample_stream_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int r = blockIdx.x / cl.num_blocks();
  // (with the wait in stream_row(): every CTA of the cluster runs before its shared memory is written)
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  stream_row<DT, GREEDY>(a, cl, sh, slice_of<DT, false>(a, cl, r, nullptr), row_state(a.temperature_s, 1.f, 0.f),
                         a.noise + r * a.noise_stride, r, dyn);
}

template <int DT, bool HELD>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int VE = Slice<DT, HELD>::VE;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, rank = (int)cl.block_rank(), nblocks = (int)cl.num_blocks();
  const int r = blockIdx.x / nblocks;
  unsigned long long* list = reinterpret_cast<unsigned long long*>(dyn);
  float* ahead = reinterpret_cast<float*>(dyn + kList * 8);
  uint4* held = reinterpret_cast<uint4*>(dyn + kListBytes);

  // (with the wait below: every CTA of the cluster runs before its shared memory is written)
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");

  // settings
  const float heat = a.temperature != nullptr ? a.temperature[r] : a.temperature_s;
  const int k_set = a.top_k != nullptr ? a.top_k[r] : a.top_k_s;
  RowState row = row_state(heat, a.top_p != nullptr ? a.top_p[r] : a.top_p_s, a.min_p != nullptr ? a.min_p[r] : a.min_p_s);
  Slice<DT, HELD> sl = slice_of<DT, HELD>(a, cl, r, held);
  const float* noise = a.noise + r * a.noise_stride;
  const bool use_k = k_set > 0 && k_set < a.vocab;
  const bool use_p = !(row.top_p >= 1.f);
  const bool single = takes_largest(heat, k_set, row.top_p, row.min_p);
  if (single || (!use_k && !use_p && !(row.min_p > 0.f))) {
    const Slice<DT, false> all = slice_of<DT, false>(a, cl, r, nullptr);
    if (single)
      stream_row<DT, true>(a, cl, sh, all, row, noise, r, dyn);
    else
      stream_row<DT, false>(a, cl, sh, all, row, noise, r, dyn);
    return;
  }
  if constexpr (HELD) {
    for (int j = tid; j < sl.chunks; j += kThreads) {
      if (sl.inside(j))
        copy_async<16>(held + j, sl.row + sl.index(j));
      else
        held[j] = sl.load(j);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const int need = (k_set + nblocks - 1) / nblocks;
  const bool use_list = use_k && need <= kThreads;
  sh.hist[tid] = sh.hist[tid + kThreads] = 0;
  if (tid == 0) sh.count = 0;
  // A thread reads back its own chunks only, here and below, but for tie_index().
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // the largest logit, and for top-k the CTA's bound: bit by bit from the top, 16 bits
  // bound it closely enough
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  uint32_t* maxima = reinterpret_cast<uint32_t*>(list);
  maxima[tid] = order(sl.largest());
  __syncthreads();
  if (tid < 32) {
    uint32_t m[kWarps], v = 0, low = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      m[i] = maxima[tid + 32 * i];
      v = max(v, m[i]);
    }
    if (use_list && need <= 8) {
      // few are needed: the need-th of these 32 lanes' maxima bounds them as well
      int larger = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const uint32_t u = __shfl_sync(0xffffffffu, v, i);
        larger += u > v || (u == v && i < tid);
      }
      low = __reduce_max_sync(0xffffffffu, larger == need - 1 ? v : 0u);
    }
    v = __reduce_max_sync(0xffffffffu, v);
    if (use_list && need > 8)
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t trial = low | 1u << bit;
        if (trial > v) continue;
        int c = 0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) c += m[i] >= trial;
        if (__reduce_add_sync(0xffffffffu, c) >= need) low = trial;
      }
    if (tid < nblocks) {
      Shared* to = cl.map_shared_rank(&sh, tid);
      to->top_of[rank] = v;
      to->bound_of[rank] = low & 0xFFFF0000u;
    }
  }
  cl.sync();
  uint32_t top = 0, low = 0xffffffffu;
  for (int q = 0; q < nblocks; ++q) {
    top = max(top, sh.top_of[q]);
    low = min(low, sh.bound_of[q]);
  }
  row.top = unorder(top);
  float bound = unorder(max(low, kLowest));
  if (row.top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs != nullptr) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  if (row.top == INFINITY) {
    sl.to_infinite();
    row.top = bound = 0.f;
  }

  // Each path leaves the CTA's best token (as pack() has it) and its part of the sum of
  // all weights in thread 0.
  unsigned long long best = 0;
  double part = 0;
  const bool want_sum = a.logprobs != nullptr;
  bool done = false;
  if (use_list) {
    float s[1] = {0.f};
    for (int j = tid; j < sl.chunks; j += kThreads) {
      if (!want_sum && !(sl.highest(j) >= bound)) continue;
      float x[VE];
      sl.get(j, x);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        if (want_sum) s[0] += row.weight(x[i]);
        if (x[i] >= bound) {
          gather(sh, list, x[i], sl.index(j) + i);
          prefetch_l2(noise + sl.index(j) + i);
        }
      }
    }
    if (want_sum) block_sum(sh, s);
    part = sh.row_sums[0];
    const int n = exchange_parts(cl, sh);
    if (n <= kFew) {
      // CTA 0 alone: it gets the candidates and counts for each the larger ones and their
      // weight, two threads a candidate. Weights are whole numbers here, as the
      // candidates come in any order.
      done = true;
      __syncthreads();   // part_start
      unsigned long long* to = cl.map_shared_rank(list + kFew, 0);
      for (int i = tid; i < (int)sh.count; i += kThreads) to[sh.part_start[rank] + i] = list[i];
      if (leave(cl, sh, 0, part)) return;
      unsigned long long* weights = reinterpret_cast<unsigned long long*>(ahead);
      const int me = tid >> 1, side = tid & 1;
      unsigned long long v = 0, w = 0, before = 0;
      float e = 1.f;
      if (me < n) {
        v = list[kFew + me];
        w = (unsigned long long)(row.weight(unorder((uint32_t)(v >> 32))) * 0x1p40f);
        e = noise[(int)~(uint32_t)v];
        if (side == 0) weights[me] = w;
      }
      __syncthreads();
      int place = 0;
      if (me < n)
#pragma unroll 4
        for (int i = side; i < n; i += 2) {
          const bool larger = list[kFew + i] > v;
          place += larger;
          before += larger ? weights[i] : 0ull;
        }
      place += __shfl_xor_sync(0xffffffffu, place, 1);
      before += __shfl_xor_sync(0xffffffffu, before, 1);
      const bool in = me < n && place < k_set;
      bool kept = in;
      if (use_p) {
        // the weight of the first k: what is before the last of them, and its own
        const int last = min(n, k_set) - 1;
        if (in && place == last && side == 0) sh.out_best = before + w;
        __syncthreads();
        kept = in && (double)before < (double)row.top_p * (double)sh.out_best;
      }
      const float z = row.z(unorder((uint32_t)(v >> 32)));
      if (row.min_p > 0.f) kept = kept && expf(z) >= row.min_p;
      kept = in && (kept || place == 0);
      best = block_best(sh, kept && z > -INFINITY ? (unsigned long long)order(race_score(z, e)) << 32 | (uint32_t)v
                                                  : 0ull);
      if (tid == 0) sh.best_of[0] = best;
    } else if (n <= kList && largest_part(sh, nblocks) <= kBins) {
      done = true;
      merge_lists(cl, sh, row, list, ahead);
      // the weight before each of this CTA's candidates, -1 past the k-th, and the weight of
      // the first k: what is before the last of them, and its own
      float* weight_before = reinterpret_cast<float*>(sh.hist);
      const int last = min(n, k_set) - 1;
      for_places(sh, list, ahead, rank, nblocks, [&](int i, unsigned long long v, int place, float before) {
        weight_before[i] = place < k_set ? before : -1.f;
        if (place != last || !use_p) return;
        const double share = (double)before + (double)row.weight(unorder((uint32_t)(v >> 32)));
        for (int q = 0; q < nblocks; ++q) cl.map_shared_rank(&sh, q)->share = share;
      });
      float target = INFINITY;
      if (use_p) {
        cl.sync();
        target = (float)((double)row.top_p * sh.share);
      } else {
        __syncthreads();
      }
      const int start = sh.part_start[rank], own = sh.part_start[rank + 1] - start;
      for (int i = tid; i < own; i += kThreads) {
        const float before = weight_before[i];
        if (!(before >= 0.f)) continue;
        const unsigned long long v = list[start + i];
        const float e = noise[(int)~(uint32_t)v], z = row.z(unorder((uint32_t)(v >> 32)));
        // nothing is before the first one alone
        if (before == 0.f || (z > -INFINITY && before < target && expf(z) >= row.min_p))
          best = max(best, (unsigned long long)order(race_score(z, e)) << 32 | (uint32_t)v);
      }
      best = block_best(sh, best);
      cl.sync();   // the lists and part weights were read
      if (leave(cl, sh, best, part)) return;
    } else {
      cl.sync();   // the counts were read
      if (tid == 0) sh.count = 0;
      __syncthreads();
    }
  }
  if (!done) {
    Cut cut = {-kFloatMax, kAnyIndex};
    bool have_sum = false;
    double whole = 0;
    if (use_k) {
      const Found f = search<DT, HELD, false>(cl, sh, sl, row, (double)k_set, cut);
      cut.x = unorder(f.key);
      if (f.single && f.above + (double)f.count > (double)k_set)
        cut.last = tie_index(cl, sh, sl, cut.x, (unsigned)((double)k_set - f.above));
    }
    if (use_p) {
      have_sum = !use_k;
      if (use_k || !nucleus(cl, sh, sl, row, list, ahead, whole, cut)) {
        // the weight of what is left, by counting
        cl.sync();
        sh.hist[tid] = sh.hist[tid + kThreads] = 0;
        __syncthreads();
        double left[1] = {whole};
        if (use_k) {
          float s[1] = {0.f};
          for (int j = tid; j < sl.chunks; j += kThreads) {
            float x[VE];
            sl.get(j, x);
#pragma unroll
            for (int i = 0; i < VE; ++i)
              if (cut.keeps(x[i], (int)sl.index(j) + i)) s[0] += row.weight(x[i]);
          }
          cluster_sum(cl, sh, s, left);
        }
        const double target = (double)row.top_p * left[0];
        const Found f = search<DT, HELD, true>(cl, sh, sl, row, target, cut);
        const float x = fmaxf(unorder(f.key), cut.x);
        int last = x > cut.x ? kAnyIndex : cut.last;
        if (f.single && f.count > 0) {
          const double part = ceil((target - f.above) / (double)row.weight(x));
          if (part < (double)f.count) last = min(last, tie_index(cl, sh, sl, x, (unsigned)max(1.0, part)));
        }
        cut.x = x;
        cut.last = last;
      }
    }
    if (row.min_p > 0.f) {
      const float x = min_p_logit(row);
      if (x > cut.x) {
        cut.x = x;
        cut.last = kAnyIndex;
      }
    }
    const bool sum_here = want_sum && !have_sum;
    float s[1] = {0.f};
    best = block_best(sh, race(sh, sl, row, cut, noise, sum_here, s[0]));
    if (sum_here) block_sum(sh, s, 3);
    part = sum_here ? sh.row_sums[3] : rank == 0 ? whole : 0.0;
    if (leave(cl, sh, best, part)) return;
  }
  finish(a, sh, sl, row, r, nblocks);
}

// A launch of clusters of n CTAs, one a row.
cudaError_t launch_clusters(void (*kernel)(SampleArgs), const SampleArgs& a, int n, int smem, cudaStream_t stream) {
  if ((int64_t)a.rows * n > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * n));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = n;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e == cudaSuccess) count_launch();
  return e;
}

template <int DT> cudaError_t launch_dt(const SampleArgs& a, int num_sms, cudaStream_t stream) {
  constexpr int VE = Slice<DT, true>::VE;
  // what all rows' settings say, where they are given for all
  const bool known = a.temperature == nullptr && a.top_k == nullptr && a.top_p == nullptr && a.min_p == nullptr;
  const bool greedy = takes_largest(a.temperature_s, a.top_k_s, a.top_p_s, a.min_p_s);
  const bool open = (a.top_k_s <= 0 || a.top_k_s >= a.vocab) && a.top_p_s >= 1.f && !(a.min_p_s > 0.f);
  if (known && (greedy || open)) {
    // the shortest sum of waves of CTAs, what a CTA does besides reading its part counting as
    // 150 KB (clusters of 1, 4 and 8: 64 rows of 151936 float32 32.1, 18.9 and 24.7 us; of 1 and
    // 8: 200 rows of bf16 44 and 59 us, one row 24.4 and 8.3 us)
    const int64_t bytes = (int64_t)a.vocab * ((DT == DT_F32 ? 4 : 2) + (greedy ? 0 : 4));
    int n = 1;
    int64_t least = INT64_MAX;
    for (int m = 1; m <= kMaxCluster; m *= 2) {
      const int64_t cost = ((int64_t)a.rows * m + 2 * num_sms - 1) / (2 * num_sms) * (150 * 1024 + bytes / m);
      if (cost < least) {
        least = cost;
        n = m;
      }
    }
    auto kernel = greedy ? sample_stream_kernel<DT, true> : sample_stream_kernel<DT, false>;
    static std::atomic<uint64_t> allowed[2];
    const cudaError_t e = allow_shared(reinterpret_cast<const void*>(kernel), kStreamBytes<DT>, allowed[greedy]);
    if (e != cudaSuccess) return e;
    return launch_clusters(kernel, a, n, kStreamBytes<DT>, stream);
  }
  const int64_t chunks = ((int64_t)a.vocab + 2 * VE - 2) / VE;   // of a row at any alignment
  // The smallest cluster that holds a row with two CTAs an SM (one computes while the
  // other loads), larger while the GPU has room for more CTAs (their steps get shorter);
  // a row past that is held by one CTA an SM, or read again each time.
  int n = 1;
  while (n < kMaxCluster && (chunks + n - 1) / n * 16 > kSliceTwo) n *= 2;
  while (n < kMaxCluster && (int64_t)a.rows * n * 2 <= 2 * num_sms) n *= 2;
  const int64_t per = (chunks + n - 1) / n;
  const bool held = per * 16 <= kSliceOne;
  const int smem = std::max(kListBytes + (held ? (int)per * 16 : 0), kStreamBytes<DT>);
  auto kernel = held ? sample_kernel<DT, true> : sample_kernel<DT, false>;
  static std::atomic<uint64_t> allowed[2];
  cudaError_t e = allow_shared(reinterpret_cast<const void*>(kernel),
                               std::max(kListBytes + (held ? kSliceOne : 0), kStreamBytes<DT>), allowed[held]);
  if (e != cudaSuccess) return e;
  return launch_clusters(kernel, a, n, smem, stream);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int dt, int num_sms, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  if (dt == DT_BF16) return launch_dt<DT_BF16>(a, num_sms, stream);
  if (dt == DT_F16) return launch_dt<DT_F16>(a, num_sms, stream);
  return launch_dt<DT_F32>(a, num_sms, stream);
}

}  // namespace fpv2
