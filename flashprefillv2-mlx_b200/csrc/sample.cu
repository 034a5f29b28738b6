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
// A row is read from DRAM once, into the shared memory of a cluster of 1 to 8 CTAs,
// and noise is read only where a token is still in the running, so the logits' bytes
// bound large batches and the chain of cluster-wide steps bounds single rows.
//
// Nothing is sorted but short lists. Top-k: every thread knows the largest logit of
// its share; the (k / CTAs)-th largest of a CTA's 1024 such values is a bound that at
// least k logits reach, and hardly more, so the few logits past it are gathered and
// sorted. Otherwise (top-p alone, k too large, too many equal logits) the threshold is
// found by counting: 1024 bins linear in x over the 32 T below the maximum, where all
// the weight is, then bins over the ordered bit patterns inside the crossing bin until
// it holds one value. Bin counts are integers and sums run in a fixed order, so a call
// repeats bit for bit.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace fpv2 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kBins = 1024;
constexpr int kList = 4096;                  // gathered candidates of a row
constexpr int kSliceBytes = 160 * 1024;      // logits a CTA holds
constexpr int kMaxCluster = 8;
constexpr uint32_t kLowest = 0x00800000u;    // order() of -FLT_MAX

// Bit patterns in the order of the floats they hold.
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unorder(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// One row's slice in a CTA: chunks of 16 bytes, aligned in memory, so the first and
// the last chunk of a row may be partly outside it (filled with -inf).
template <int DT> struct Slice {
  static constexpr int VE = DT == DT_F32 ? 4 : 8;
  using T = typename Elem<DT>::T;
  const T* row;
  const uint4* held;   // shared memory, null when the slice is read from global each time
  int64_t first;       // index of the first element of chunk 0 (may be negative)
  int chunks, vocab;

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
  // the chunk as floats: NaN as -inf, -0 as +0
  __device__ __forceinline__ void get(int j, float (&x)[VE]) const {
    const uint4 u = held != nullptr ? held[j] : load(j);
    const uint32_t r[4] = {u.x, u.y, u.z, u.w};
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<DT>(r[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = fmaxf(x[i], -INFINITY) + 0.f;
  }
};

struct Shared {
  unsigned hist[kBins];
  unsigned long long best[32];
  double sums[32][4];
  // written by this CTA, read by the cluster
  unsigned long long row_best, row_race;
  double row_sums[4];
  unsigned count, bound, ties;
  // broadcast inside the CTA
  unsigned long long out_best;
  double out_sums[4];
  double scan[32];
  unsigned found_bin, found_count;
  double found_above;
  int tie_last;
};

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}

// Largest of `v` over the cluster, in every thread.
__device__ unsigned long long cluster_max(cg::cluster_group& cl, Shared& sh, unsigned long long v,
                                          unsigned long long Shared::*slot) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) sh.best[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = warp_max(sh.best[threadIdx.x]);
    if (threadIdx.x == 0) sh.*slot = v;
  }
  cl.sync();
  if (threadIdx.x == 0) {
    v = 0;
    for (unsigned r = 0; r < cl.num_blocks(); ++r) {
      const unsigned long long u = *cl.map_shared_rank(&(sh.*slot), r);
      v = u > v ? u : v;
    }
    sh.out_best = v;
  }
  __syncthreads();
  return sh.out_best;
}

// Sums of N values over the cluster, in a fixed order, in every thread.
template <int N> __device__ void cluster_sum(cg::cluster_group& cl, Shared& sh, double (&v)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (lane == 0) sh.sums[warp][i] = v[i];
  }
  cl.sync();   // also: the last read of row_sums is over
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double s = sh.sums[lane][i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) sh.row_sums[i] = s;
    }
  }
  cl.sync();
  if (threadIdx.x < N) {
    double s = 0;
    for (unsigned r = 0; r < cl.num_blocks(); ++r) s += cl.map_shared_rank(&sh, r)->row_sums[threadIdx.x];
    sh.out_sums[threadIdx.x] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = sh.out_sums[i];
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
    const double mine = sh.scan[lane];
    double s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    sh.scan[lane] = s - mine;
  }
  __syncthreads();
  return sh.scan[warp] + (incl - v);
}

// Descending bitonic sort of n (a power of two, at least 2) values in shared memory.
template <typename K> __device__ void sort_down(K* v, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const bool down = (lo & size) == 0;
        const K x = v[lo], y = v[hi];
        if ((x < y) == down) {
          v[lo] = y;
          v[hi] = x;
        }
      }
    }
  __syncthreads();
}

// The settings of one row and what its logits give.
struct RowState {
  float heat, inv_heat, top, scale;   // T, 1/T, the largest logit, bins per logit
  float top_p, min_p;

  __device__ __forceinline__ float z(float x) const { return x == top ? 0.f : __fdiv_rn(x - top, heat); }
  __device__ __forceinline__ float z_near(float x) const { return x == top ? 0.f : (x - top) * inv_heat; }
  __device__ __forceinline__ float weight(float x) const { return ex2(z_near(x) * kLog2e); }
  __device__ __forceinline__ int bin(float x) const {
    return x == top ? 0 : (int)fminf((top - x) * scale, (float)(kBins - 1));
  }
};

// A threshold: keys above `key`, and of those equal to it the ones up to index `last`.
struct Cut {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool keeps(uint32_t k, int64_t at) const {
    return k > key || (k == key && at <= last);
  }
};

// Adds up the bins of the cluster's CTAs; thread i gets bin i.
__device__ unsigned gather_bin(cg::cluster_group& cl, Shared& sh) {
  cl.sync();
  unsigned c = 0;
  for (unsigned r = 0; r < cl.num_blocks(); ++r) c += cl.map_shared_rank(&sh, r)->hist[threadIdx.x];
  cl.sync();
  sh.hist[threadIdx.x] = 0;
  return c;
}

// Search for the value where the ordered logits reach `target` (a count, or a weight).
// On return the crossing value is `key` with `count` logits equal to it and `above` of
// the target used up by larger ones; or, when `count` logits in all are known to be
// needed, `key` is a lower bound that just these reach.
struct Found {
  uint32_t key;
  unsigned count;
  double above;
  bool single;   // `key` is one value (else a bound with all `count` logits needed)
};

template <int DT, bool WEIGHT>
__device__ Found search(cg::cluster_group& cl, Shared& sh, const Slice<DT>& sl, const RowState& row,
                        double target, const Cut& within) {
  constexpr int VE = Slice<DT>::VE;
  const int tid = threadIdx.x;
  // linear bins
  for (int j = tid; j < sl.chunks; j += kThreads) {
    float x[VE];
    sl.get(j, x);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      if (x[i] == -INFINITY || order(x[i]) < within.key) continue;
      const int b = row.bin(x[i]);
      // the last bin's weight is nothing next to the row's, and its count is what is left
      if (!WEIGHT || b < kBins - 1) atomicAdd(&sh.hist[b], 1u);
    }
  }
  unsigned c = gather_bin(cl, sh);
  double mass = (double)c;
  if (WEIGHT) mass *= (double)ex2(-((float)tid + (tid == 0 ? 0.f : 0.5f)) / row.scale * row.inv_heat * kLog2e);
  double before = block_before(sh, mass);
  if (tid == 0) sh.found_bin = kBins - 1;
  __syncthreads();
  if (before + mass >= target) atomicMin(&sh.found_bin, (unsigned)tid);
  __syncthreads();
  int bin = (int)sh.found_bin;
  double above;
  unsigned count;
  if (!WEIGHT) {
    if (tid == bin) {
      sh.found_above = before;
      sh.found_count = c;
    }
    __syncthreads();
    above = sh.found_above;
    count = sh.found_count;
  } else {
    // The bins' weights were estimates: sum the weights above and in three bins around.
    int moved = 0;
    while (true) {
      bin = min(max(bin, 1), kBins - 2);
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      for (int j = tid; j < sl.chunks; j += kThreads) {
        float x[VE];
        sl.get(j, x);
        const int64_t at = sl.index(j);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          if (x[i] == -INFINITY || !within.keeps(order(x[i]), at + i)) continue;
          const int b = row.bin(x[i]);
          if (b > bin + 1) continue;
          const float w = row.weight(x[i]);
          s[0] += b < bin - 1 ? w : 0.f;
          s[1] += b == bin - 1 ? w : 0.f;
          s[2] += b == bin ? w : 0.f;
          s[3] += b == bin + 1 ? w : 0.f;
        }
      }
      double v[4] = {s[0], s[1], s[2], s[3]};
      cluster_sum(cl, sh, v);
      if (v[0] >= target && bin > 1 && moved <= 0) {
        bin -= 3;
        moved = -1;
        continue;
      }
      if (v[0] + v[1] + v[2] + v[3] < target && bin < kBins - 2 && moved >= 0) {
        bin += 3;
        moved = 1;
        continue;
      }
      above = v[0];
      bin -= 1;
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
    count = 0xffffffffu;   // not known: the levels below count
  }
  // the keys of the bin: bin() falls as the key grows
  uint32_t lo = kLowest, hi = order(row.top);
  if (bin < kBins - 1) {   // smallest key whose bin is <= bin
    uint32_t a = kLowest, b = hi;
    while (a < b) {
      const uint32_t mid = a + (b - a) / 2;
      if (row.bin(unorder(mid)) <= bin) b = mid; else a = mid + 1;
    }
    lo = a;
  }
  if (bin > 0) {           // largest key whose bin is >= bin
    uint32_t a = lo, b = hi;
    while (a < b) {
      const uint32_t mid = a + (b - a + 1) / 2;
      if (row.bin(unorder(mid)) >= bin) a = mid; else b = mid - 1;
    }
    hi = a;
  }
  if (lo < within.key) lo = within.key;
  if (hi < lo) return {lo, 0, above, false};   // the target is just past all there is
  while (true) {
    if (!WEIGHT && above + (double)count <= target) return {lo, count, above, false};
    if (count == 1) return {lo, 1, above, false};
    if (lo >= hi && count != 0xffffffffu) return {lo, count, above, true};
    const uint32_t width = hi - lo;   // keys less one
    const int bits = 32 - __clz(width | 1), shift = bits > 10 ? bits - 10 : 0;
    for (int j = tid; j < sl.chunks; j += kThreads) {
      float x[VE];
      sl.get(j, x);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const uint32_t k = order(x[i]);
        if (k >= lo && k <= hi) atomicAdd(&sh.hist[(hi - k) >> shift], 1u);
      }
    }
    c = gather_bin(cl, sh);
    mass = (double)c;
    const uint32_t off = (uint32_t)tid << shift;
    if (WEIGHT && c != 0) {
      // a bin of several values weighs as its middle one: it spans under 2^-15 of z
      const uint32_t span = (1u << shift) - 1;
      const uint32_t mid = hi - off - min(span / 2, (hi - off - lo) / 2);
      mass *= (double)row.weight(unorder(mid));
    }
    before = block_before(sh, mass) + above;
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
    const unsigned at = sh.found_bin;
    if (tid == (int)at) {
      sh.found_above = before;
      sh.found_count = c;
    }
    __syncthreads();
    above = sh.found_above;
    count = sh.found_count;
    hi = hi - (at << shift);
    const uint32_t span = (1u << shift) - 1;
    if (hi - lo > span) lo = hi - span;
    __syncthreads();
  }
}

// Index of the `need`-th logit (from 1) equal to `key`, in index order.
template <int DT>
__device__ int tie_index(cg::cluster_group& cl, Shared& sh, const Slice<DT>& sl, uint32_t key, unsigned need) {
  constexpr int VE = Slice<DT>::VE;
  const int share = (sl.chunks + kThreads - 1) / kThreads;   // chunks a thread, consecutive
  const int j0 = min(sl.chunks, (int)threadIdx.x * share), j1 = min(sl.chunks, j0 + share);
  unsigned mine = 0;
  for (int j = j0; j < j1; ++j) {
    float x[VE];
    sl.get(j, x);
#pragma unroll
    for (int i = 0; i < VE; ++i) mine += order(x[i]) == key;
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
        if (order(x[i]) == key && ++seen == need) {
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

__device__ __forceinline__ unsigned long long pack(uint32_t key, int64_t at) {
  return (unsigned long long)key << 32 | (uint32_t)~(uint32_t)at;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleArgs a, int per) {
  using T = typename Elem<DT>::T;
  constexpr int VE = Slice<DT>::VE;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Shared sh;
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, rank = (int)cl.block_rank(), nblocks = (int)cl.num_blocks();
  const int r = blockIdx.x / nblocks;
  unsigned long long* list = reinterpret_cast<unsigned long long*>(dyn);
  uint4* held = reinterpret_cast<uint4*>(dyn + kList * 8);

  Slice<DT> sl;
  sl.row = reinterpret_cast<const T*>(a.logits) + r * a.logits_stride;
  sl.vocab = a.vocab;
  const int mis = (int)(reinterpret_cast<uintptr_t>(sl.row) % 16 / sizeof(T));
  const int all = (int)(((int64_t)mis + a.vocab + VE - 1) / VE);
  const int share = (all + nblocks - 1) / nblocks;   // <= per when slices are held
  const int c0 = min(all, rank * share);
  sl.chunks = min(share, all - c0);
  sl.first = (int64_t)c0 * VE - mis;
  sl.held = nullptr;
  if (per > 0) {
    for (int j = tid; j < sl.chunks; j += kThreads) {
      if (sl.inside(j))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(held + j)),
                     "l"(sl.row + sl.index(j))
                     : "memory");
      else
        held[j] = sl.load(j);
    }
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    sl.held = held;
  }
  sh.hist[tid] = 0;
  if (tid == 0) sh.count = 0;
  __syncthreads();

  // settings
  RowState row;
  const float heat = a.temperature != nullptr ? a.temperature[r] : a.temperature_s;
  row.top_p = a.top_p != nullptr ? a.top_p[r] : a.top_p_s;
  row.min_p = a.min_p != nullptr ? a.min_p[r] : a.min_p_s;
  const int k_set = a.top_k != nullptr ? a.top_k[r] : a.top_k_s;
  const bool greedy = !(heat > 0.f);
  row.heat = greedy ? 1.f : heat;
  row.inv_heat = 1.f / row.heat;
  row.scale = (float)kBins / 32.f * row.inv_heat;

  // the largest logit and its lowest index
  float mx = -INFINITY;
  int64_t mx_at = 0;
  for (int j = tid; j < sl.chunks; j += kThreads) {
    float x[VE];
    sl.get(j, x);
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (x[i] > mx) {
        mx = x[i];
        mx_at = sl.index(j) + i;
      }
  }
  const unsigned long long top = cluster_max(cl, sh, pack(order(mx), mx_at), &Shared::row_best);
  row.top = unorder((uint32_t)(top >> 32));
  const int first = (int)~(uint32_t)top;
  if (row.top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs != nullptr) a.logprobs[r] = -INFINITY;
    }
    cl.sync();   // no CTA leaves while another may read its shared memory
    return;
  }
  const bool use_k = k_set > 0 && k_set < a.vocab;
  const bool use_p = !(row.top_p >= 1.f);
  const bool single = greedy || k_set == 1 || !(row.top_p > 0.f) || !(row.min_p <= 1.f);

  double whole = 0;   // sum of all weights
  if (a.logprobs != nullptr || (!single && use_p && !use_k)) {
    float s = 0.f;
    for (int j = tid; j < sl.chunks; j += kThreads) {
      float x[VE];
      sl.get(j, x);
#pragma unroll
      for (int i = 0; i < VE; ++i) s += x[i] == -INFINITY ? 0.f : row.weight(x[i]);
    }
    double v[1] = {s};
    cluster_sum(cl, sh, v);
    whole = v[0];
  }

  int token = first;
  if (!single) {
    const float* noise = a.noise + r * a.noise_stride;
    bool done = false;
    Cut cut = {0, 0};
    if (use_k && (k_set + nblocks - 1) / nblocks <= kThreads) {
      // bound that at least k logits reach
      uint32_t* maxima = reinterpret_cast<uint32_t*>(list);
      maxima[tid] = order(mx);
      sort_down(maxima, kThreads);
      if (tid == 0) sh.bound = maxima[(k_set + nblocks - 1) / nblocks - 1];
      cl.sync();
      uint32_t bound = 0xffffffffu;
      for (int q = 0; q < nblocks; ++q) bound = min(bound, cl.map_shared_rank(&sh, q)->bound);
      for (int j = tid; j < sl.chunks; j += kThreads) {
        float x[VE];
        sl.get(j, x);
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (x[i] > -INFINITY && order(x[i]) >= bound) {
            const unsigned at = atomicAdd(&sh.count, 1u);
            if (at < kList) list[at] = pack(order(x[i]), sl.index(j) + i);
          }
      }
      cl.sync();
      unsigned n = 0, before = 0;
      for (int q = 0; q < nblocks; ++q) {
        const unsigned c = cl.map_shared_rank(&sh, q)->count;
        if (q < rank) before += c;
        n += c;
      }
      if (n <= kList) {
        done = true;
        if (rank != 0) {   // hand the candidates to CTA 0
          unsigned long long* to = cl.map_shared_rank(list, 0);
          for (unsigned i = tid; i < sh.count; i += kThreads) to[before + i] = list[i];
        }
        cl.sync();
        if (rank == 0) {
          int n2 = 2;
          while (n2 < (int)n) n2 <<= 1;
          for (int i = (int)n + tid; i < n2; i += kThreads) list[i] = 0;
          sort_down(list, n2);
          const int kept = min((int)n, k_set);
          constexpr int EACH = kList / kThreads;
          float w[EACH];
          double mine = 0;
#pragma unroll
          for (int i = 0; i < EACH; ++i) {
            const int at = tid * EACH + i;
            w[i] = at < kept ? expf(row.z(unorder((uint32_t)(list[at] >> 32)))) : 0.f;
            mine += w[i];
          }
          double run = block_before(sh, mine);
          if (tid == kThreads - 1) sh.found_above = run + mine;
          __syncthreads();
          const double target = use_p ? (double)row.top_p * sh.found_above : INFINITY;
          unsigned long long best = 0;
#pragma unroll
          for (int i = 0; i < EACH; ++i) {
            const int at = tid * EACH + i;
            if (at < kept && (at == 0 || (run < target && w[i] >= row.min_p))) {
              const float z = row.z(unorder((uint32_t)(list[at] >> 32)));
              const int id = (int)~(uint32_t)list[at];
              if (z > -INFINITY) {
                const unsigned long long v = pack(order(race_score(z, noise[id])), id);
                best = v > best ? v : best;
              }
            }
            run += w[i];
          }
          best = warp_max(best);
          if ((tid & 31) == 0) sh.best[tid >> 5] = best;
          __syncthreads();
          if (tid < 32) {
            best = warp_max(sh.best[tid]);
            token = (int)~(uint32_t)best;
          }
        }
      }
    }
    if (!done) {
      if (use_k) {
        const Found f = search<DT, false>(cl, sh, sl, row, (double)k_set, Cut{0, 0});
        cut.key = f.key;
        cut.last = 0x7fffffff;
        if (f.single && f.above + (double)f.count > (double)k_set)
          cut.last = tie_index(cl, sh, sl, f.key, (unsigned)((double)k_set - f.above));
      }
      if (use_p) {
        double weight = whole;
        if (use_k) {
          float s = 0.f;
          for (int j = tid; j < sl.chunks; j += kThreads) {
            float x[VE];
            sl.get(j, x);
#pragma unroll
            for (int i = 0; i < VE; ++i)
              if (x[i] > -INFINITY && cut.keeps(order(x[i]), sl.index(j) + i)) s += row.weight(x[i]);
          }
          double v[1] = {s};
          cluster_sum(cl, sh, v);
          weight = v[0];
        } else {
          cut.last = 0x7fffffff;
        }
        const double target = (double)row.top_p * weight;
        const Found f = search<DT, true>(cl, sh, sl, row, target, cut);
        int last = f.key > cut.key ? 0x7fffffff : cut.last;
        if (f.single) {
          const double need = ceil((target - f.above) / (double)row.weight(unorder(f.key)));
          if (need < (double)f.count) {
            const int at = tie_index(cl, sh, sl, f.key, (unsigned)max(1.0, need));
            last = min(last, at);
          }
        }
        cut.key = f.key;
        cut.last = last;
      }
      // the race over what is left
      const bool all_kept = !use_k && !use_p;
      float best = -INFINITY;
      unsigned long long best_key = 0;
      for (int j = tid; j < sl.chunks; j += kThreads) {
        float x[VE];
        sl.get(j, x);
        const int64_t at = sl.index(j);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          if (!(x[i] > -INFINITY)) continue;
          if (!all_kept && !cut.keeps(order(x[i]), at + i)) continue;
          if (row.min_p > 0.f && at + i != first && !(expf(row.z(x[i])) >= row.min_p)) continue;
          const float e = noise[at + i];
          // the exact score only where a near one could win
          if (row.z_near(x[i]) - __logf(e) < best - 2e-3f) continue;
          const float z = row.z(x[i]);
          if (!(z > -INFINITY)) continue;
          const float s = race_score(z, e);
          const unsigned long long v = pack(order(s), at + i);
          if (v > best_key) {
            best_key = v;
            best = s;
          }
        }
      }
      token = (int)~(uint32_t)cluster_max(cl, sh, best_key, &Shared::row_race);
    }
  }
  if (rank == 0 && tid == 0) {
    a.tokens[r] = token;
    if (a.logprobs != nullptr) {
      const float x = fmaxf(Elem<DT>::to_f(sl.row[token]), -INFINITY) + 0.f;
      a.logprobs[r] = row.z(x) - (float)log(whole);
    }
  }
  cl.sync();
}

template <int DT> cudaError_t launch_dt(const SampleArgs& a, int num_sms, cudaStream_t stream) {
  constexpr int VE = Slice<DT>::VE;
  const int64_t chunks = ((int64_t)a.vocab + 2 * VE - 2) / VE;   // of a row at any alignment
  // the smallest cluster that holds a row, larger while the GPU has CTAs to spare
  int n = 1;
  while (n < kMaxCluster && (chunks + n - 1) / n * 16 > kSliceBytes) n *= 2;
  while (n < kMaxCluster && (int64_t)a.rows * n * 2 <= num_sms) n *= 2;
  const int64_t per = (chunks + n - 1) / n;
  const bool held = per * 16 <= kSliceBytes;
  const int smem = kList * 8 + (held ? (int)per * 16 : 0);
  cudaError_t e = cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kList * 8 + kSliceBytes);
  if (e != cudaSuccess) return e;
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
  e = cudaLaunchKernelEx(&cfg, sample_kernel<DT>, a, held ? (int)per : 0);
  if (e == cudaSuccess) count_launch();
  return e;
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int dt, int num_sms, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  if (dt == DT_BF16) return launch_dt<DT_BF16>(a, num_sms, stream);
  if (dt == DT_F16) return launch_dt<DT_F16>(a, num_sms, stream);
  return launch_dt<DT_F32>(a, num_sms, stream);
}

}  // namespace fpv2
