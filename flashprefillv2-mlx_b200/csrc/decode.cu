// Attention of the newest token (or the newest few) of every sequence over its
// paged K/V.
//
// Row t of sequence b sits at position p = len_b - T + t and sees key j when
// j <= p and (j < sinks or j > p - window); window 0 sees all j <= p.
//   o = sum_j softmax_j(scale q.k_j) v_j,   lse = log sum_j exp(scale q.k_j)
// A row that sees nothing gets o = 0 and lse = -inf.
//
// Every visible K and V row takes 4 G T D operations on 4 D bytes, so DRAM bandwidth
// bounds the call while few rows share a KV head; the tensor work is small and a few
// rows wide, so it runs on mma.sync m16n8k16 straight from shared memory, without TMEM
// round trips. A tile is fetched once for each group of up to 16 rows (32 for head_dim 64),
// by warps of their own, so past that the time grows with the groups (16 sequences of 8000
// keys, 8 KV heads of 128, 80 us at a copy's rate: up to 8 rows 98 us, 16 106, 32 156, 64 294).
//
// Split: the visible keys of all sequences are one stream of TK-key tiles, cut
// into equal parts whatever the sequences' lengths are. One warp takes one part
// for one KV head (and up to 32 of its query rows), with its own cp.async ring
// and running softmax, so warps never wait for each other; neighbouring warps
// take neighbouring heads of the same keys, which keeps the page reads of a
// block of threads contiguous. A sequence that lies inside one part is finished
// there; the pieces of the others go to the workspace in float32 and a second
// kernel, launched early and waiting for the first, joins them in part order, so
// the result does not depend on timing.
//
// Measured (bf16, 32 + 8 heads of 128): 64 sequences of 129 to 16384 keys 177 us for 975 MB
// (means of three draws), 5.5 TB/s, 0.84 of a copy; one of 65536 keys 54 us, 5.0 TB/s (50 us without
// the join), of which about 3 us pass before the first keys are asked for and 8 us while the last
// warps finish; one of 517 keys 8.2 us, latency.
#include "common.cuh"
#include "kernels.h"

namespace fpv2 {
namespace {

constexpr int kSms = 148;      // B200; sets the split, so results do not vary with the device
constexpr float kLn2 = 0.6931471805599453f;

// Keys a tile, ring stages, warps a CTA (about 200 KB of ring). Measured when they were chosen,
// head_dim 128, one sequence of 65536 keys and a ragged batch of 64: {16, 3, 8} 56.3 and 175 us,
// {16, 6, 4} 58.5 and 170, {16, 5, 5} 56.7 and 189, {16, 2, 12} 62 and 173, {32, 2, 6} 64.6 and 166,
// {32, 3, 4} 80 and 167. The others by 16 sequences of 8000 keys in pages of 16, 8 KV heads: 64: {32,
// 3, 8} 57.4 us, {16, 6, 8} 56.5, {32, 4, 6} 69.7, the first with half the steps for compute.
// 96: {16, 4, 8} 76.5, {16, 3, 11} 82.9, {32, 3, 5} 148. 256 (4 KV heads): {16, 3, 4} 96.9, {16, 2, 6}
// 100.3.
template <int D> struct Shape;
template <> struct Shape<64> { static constexpr int TK = 32, ST = 3, NW = 8; };
template <> struct Shape<96> { static constexpr int TK = 16, ST = 4, NW = 8; };
template <> struct Shape<128> { static constexpr int TK = 16, ST = 3, NW = 8; };
template <> struct Shape<256> { static constexpr int TK = 16, ST = 3, NW = 4; };

// Bytes between rows of a tile in shared memory: one 16-byte chunk more than the
// row, so the eight rows of an ldmatrix fall into different banks.
template <int D> constexpr int kPitch = D * 2 + 16;
template <int D> constexpr int kStageBytes = 2 * Shape<D>::TK * kPitch<D>;

// Blocks of eight query rows a warp takes, and the warps that share a KV head's rows.
// More blocks reuse a tile in shared memory but need their queries and accumulators in
// registers, 3 D / 4 a block and lane with the addresses and scores beside them: four
// blocks fit for head_dim 64 alone (at 128, 8 x 8000 keys of 32 rows a head take 203 us
// with four blocks, which spill, and 100 us with two and the tiles fetched twice).
__host__ __device__ inline int blocks_of(int rows, int D) {
  return rows <= 8 ? 1 : rows <= 16 || D > 64 ? 2 : 4;
}
__host__ __device__ inline int row_groups(int rows, int D) {
  const int per = 8 * blocks_of(rows, D);
  return (rows + per - 1) / per;
}

// The visible tiles of one sequence: tile t holds keys from (t < head ? t : t + jump) * TK.
struct Seq {
  int len, tiles, head, jump, low;   // low: first key of the widest window
};

template <int TK> __device__ __forceinline__ Seq seq_of(const DecodeArgs& a, int b) {
  Seq s;
  const int64_t room = (int64_t)a.table_width * a.page_size;
  int64_t len = b < a.B ? a.lengths[b] : 0;
  len = len < 0 ? 0 : (len > room ? room : len);
  s.len = (int)len;
  const int all = (s.len + TK - 1) / TK;
  s.tiles = all;
  s.head = all;
  s.jump = 0;
  s.low = 0;
  if (a.window > 0) {
    const int64_t low = len - a.T - (int64_t)a.window + 1;
    s.low = low > 0 ? (int)low : 0;
    const int first = s.low / TK, head = (min(a.sinks, s.len) + TK - 1) / TK;
    if (head < first) {
      s.head = head;
      s.jump = first - head;
      s.tiles = all - s.jump;
    }
  }
  return s;
}

__device__ __forceinline__ int64_t warp_sum(uint32_t v) {
  const uint32_t low = __reduce_add_sync(0xffffffffu, v & 0xffffu), high = __reduce_add_sync(0xffffffffu, v >> 16);
  return ((int64_t)high << 16) + low;
}

// A sequence costs its tiles and some more, for its queries' way in and its results' way
// out; the stream that is cut into parts counts that first, ahead of the tiles. (24
// sequences of 3 to 20011 keys, 32 rows a head: the slowest warp takes 83k cycles without it,
// 44k with two tiles' worth; in all 38.0 us with two, 34.6 with four, 33.6 with six. 40
// sequences of 9 to 900 keys, 4 rows: 17.0, 17.1 and 17.6 us.)
constexpr int kSeqCost = 4;
__device__ __forceinline__ int cost_of(const Seq& s) { return s.tiles > 0 ? s.tiles + kSeqCost : 0; }

// Stream units before sequence `want` and in total (warp-wide).
template <int TK>
__device__ __forceinline__ void scan_to(const DecodeArgs& a, int lane, int want, int64_t& before,
                                        int64_t& total) {
  before = total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const uint32_t n = cost_of(seq_of<TK>(a, b0 + lane));
    if (want > b0) before += warp_sum(b0 + lane < want ? n : 0u);
    total += warp_sum(n);
  }
}

// a / b for non-negative a and positive b, mostly of 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// Stream units a part. Not fewer than balances what a tile adds to the first kernel (about
// 1000 cycles) with what a piece adds to the second (about 5: eight warps, 24 in flight each):
// the square root of total / 200. It matters with few KV heads, where one wave of warps is
// many parts (6 rows on one KV head of 128: 60000 keys 15.8 us, 64 sequences of 60 to 4000
// 21.4 us; by total / 90 17.3 and 23.3, by total / 40 19.4 and 27.3).
__device__ __forceinline__ int64_t part_tiles(int64_t total, int parts) {
  return max(quotient(total + parts - 1, parts), (int64_t)sqrtf((float)total * (1.f / 200.f)));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_if(uint32_t dst, const void* src, bool read) {
  const int n = read ? 16 : 0;   // 0: the chunk is filled with zeros and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// 8 x 8 transpose of 16-bit values spread over the warp.
__device__ __forceinline__ uint32_t turn(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// c += a b for a 16 x 16 by 16 x 8 tile.
template <int DT>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == DT_BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Walks the tiles of a part: sequence, tile in it, and the tile's place in the stream.
template <int TK> struct Walk {
  int b, t;
  Seq s;
  int64_t at;

  __device__ __forceinline__ void next(const DecodeArgs& a, int64_t end) {
    ++t;
    ++at;
    while (t >= s.tiles && at + kSeqCost < end) {   // a sequence with tiles ahead
      ++b;
      s = seq_of<TK>(a, b);
      if (s.tiles > 0) {
        t = 0;
        at += kSeqCost;
      }
    }
    if (t >= s.tiles) at = end;
  }
};

// The walk for the copies, with this lane's row of the tile: its page (loaded one tile
// before it is needed) and place in the page.
template <int TK> struct Feed : Walk<TK> {
  using Walk<TK>::b;
  using Walk<TK>::t;
  using Walk<TK>::s;
  int page, in_page;

  __device__ __forceinline__ int key0() const { return (t < s.head ? t : t + s.jump) * TK; }
  __device__ __forceinline__ void fetch(const DecodeArgs& a, int lane, bool whole) {
    // every lane of a tile inside one page: its first row; past the end: the last key
    const int key = min(key0() + (whole ? 0 : lane % TK), s.len - 1);
    const int at = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
    in_page = key - at * a.page_size;
    page = a.tables[(int64_t)b * a.table_stride + at];
  }
};

// Scores are taken transposed, S^T = K Q^T with 16 keys by 8 query rows a product, so a
// GQA group of up to eight rows fills the tile, and O^T = V^T P^T likewise; P^T comes
// from S^T's registers by an 8 x 8 transpose.
// Registers: a CTA of 256 threads with 192 leaves a CTA of the second kernel its 16384.
template <int D, int NB> constexpr int kRegs = NB <= 2 && D < 256 ? 192 : 255;

template <int DT, int D, int NB>
__global__ void __maxnreg__((kRegs<D, NB>)) decode_kernel(const DecodeArgs a, int parts) {
  constexpr int TK = Shape<D>::TK, ST = Shape<D>::ST, NW = Shape<D>::NW;
  constexpr int PITCH = kPitch<D>, CH = D / 8, KS = D / 16, MT = TK / 16;
  constexpr int CL = CH <= 8 ? 8 : CH <= 16 ? 16 : 32;   // lanes that copy one row
  constexpr int RPS = 32 / CL;                           // rows a warp-wide copy covers
  // P is 2^(score - m) for an m that lies kLift below the largest score it was set from and is
  // only moved when one passes it by kLift + kSlack. float16 goes up to 2^16 and down to 2^-24:
  // lifted by 7 a weight is held to 2^-32 of the largest one, which keeps a long tail of small
  // ones (at 2^-25, 32768 keys of 2^-25 each came out as nothing). bfloat16 has no such end.
  constexpr float kSlack = 8.f, kLift = DT == DT_F16 ? 7.f : 0.f;
  using T = typename Elem<DT>::T;
  extern __shared__ __align__(16) unsigned char smem[];
  // launched while the kernel before it in the stream still runs: wait for its results
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;   // mma fragments: rows g and g + 8, column pair c
  const int R = a.G * a.T;                 // query rows of a KV head
  const int groups = row_groups(R, D), cols = a.Hkv * groups;
  const unsigned wi = blockIdx.x * NW + warp;
  const int part = (int)(wi / (unsigned)cols), col = (int)(wi - (unsigned)part * cols);
  const int h = col / groups, rbase = (col - h * groups) * 8 * NB;
  if (part >= parts) return;

  // this warp's range of the tile stream, and the sequence it starts in
  int64_t unused, total;
  scan_to<TK>(a, lane, 0, unused, total);
  const int64_t chunk = part_tiles(total, parts);
  const int64_t begin = (int64_t)part * chunk, end = min(begin + chunk, total);
  if (begin >= end) return;
  const bool whole = a.page_size % TK == 0;
  Feed<TK> f;
  bool started;   // the first sequence started in an earlier part
  {
    int64_t run = 0;
    int b0 = 0;
    while (true) {
      const uint32_t n = cost_of(seq_of<TK>(a, b0 + lane));
      if (b0 + 32 < a.B) {   // (the last 32 hold it if those before do not)
        const int64_t sum = warp_sum(n);
        if (run + sum <= begin) {
          run += sum;
          b0 += 32;
          continue;
        }
      }
      uint32_t ahead = n;   // units of the lanes before this one; less than 32 (2^27 + 2)
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, ahead, o);
        if (lane >= o) ahead += v;
      }
      ahead -= n;
      const int at = 31 - __clz(__ballot_sync(0xffffffffu, n > 0 && (int64_t)ahead <= begin - run));
      f.b = b0 + at;
      run += __shfl_sync(0xffffffffu, ahead, at);   // where the sequence starts
      f.t = max((int)(begin - run) - kSeqCost, 0);
      f.at = run + kSeqCost + f.t;
      started = run < begin;
      break;
    }
    f.s = seq_of<TK>(a, f.b);
  }
  if (f.at >= end) return;   // nothing but the cost of a sequence whose tiles are the next part's
  f.fetch(a, lane, whole);
  Walk<TK> w = f;    // the consumer's
  int seg0 = f.t;    // its segment's first tile

  unsigned char* const ring_ptr = smem + warp * ST * kStageBytes<D>;
  const uint32_t ring = smem_u32(ring_ptr);
  const int lrow = lane / CL, lch = lane % CL;           // this lane's row and chunk of a copy
  const T* kh = reinterpret_cast<const T*>(a.k) + h * a.k_sh + lch * 8;
  const T* vh = reinterpret_cast<const T*>(a.v) + h * a.v_sh + lch * 8;
  const uint32_t ldst = lrow * PITCH + lch * 16;
  int fill = 0;   // the ring slot of the next copy

  auto issue = [&](const Feed<TK>& f) {
    if (f.at < end) {
      const uint32_t dst = ring + fill * kStageBytes<D> + ldst;
      fill = fill + 1 == ST ? 0 : fill + 1;
      const int key0 = f.key0();
      // a page of this lane's own row may hold no key that any query sees; its entry is not reported
      const int mine = key0 + lane % TK;
      const bool used = whole || (mine < f.s.len && (mine >= f.s.low || mine < a.sinks));
      const int page = clamp_entry(f.page, 0, a.num_pages - 1, used ? a.status : nullptr);
      const int64_t ko = page * a.k_sp + f.in_page * a.k_sr, vo = page * a.v_sp + f.in_page * a.v_sr;
      const bool all = key0 + TK <= f.s.len && (key0 >= f.s.low || key0 + TK <= a.sinks);
      if (whole && all) {
        const T* kp = kh + ko + lrow * a.k_sr;
        const T* vp = vh + vo + lrow * a.v_sr;
        if (CL == CH || lch < CH) {
#pragma unroll
          for (int i = 0; i < TK / RPS; ++i) {
            cp16(dst + i * RPS * PITCH, kp);
            kp += RPS * a.k_sr;
          }
#pragma unroll
          for (int i = 0; i < TK / RPS; ++i) {
            cp16(dst + (TK + i * RPS) * PITCH, vp);
            vp += RPS * a.v_sr;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < TK / RPS; ++i) {
          const int row = lrow + i * RPS, key = key0 + row;
          const int64_t kr = whole ? ko + row * a.k_sr : __shfl_sync(0xffffffffu, ko, row);
          const int64_t vr = whole ? vo + row * a.v_sr : __shfl_sync(0xffffffffu, vo, row);
          // keys that no row sees are zeros, whatever their page holds
          const bool seen = key < f.s.len && (key >= f.s.low || key < a.sinks);
          if (CL == CH || lch < CH) {
            cp16_if(dst + i * RPS * PITCH, kh + kr, seen);
            cp16_if(dst + (TK + i * RPS) * PITCH, vh + vr, seen);
          }
        }
      }
    }
    cp_commit();
  };
  auto advance = [&]() {
    if (f.at < end) f.next(a, end);
    if (f.at < end) f.fetch(a, lane, whole);
  };
  bool careful = false;   // a segment is taken a second time, for its values' infinities
again:
  {
    Feed<TK> early[ST - 1];   // their table entries are loaded side by side
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      early[i] = f;
      advance();
    }
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) issue(early[i]);
  }

  uint32_t qf[NB][KS][2];
  float o[NB][KS][4];
  float m[NB][2], e[NB][2], l[NB][2];   // running maximum less kLift, the same with -inf as 0, sum: rows 2 c, 2 c + 1
  int tq[NB][2];                        // their new-token index
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) tq[n][j] = (rbase + n * 8 + c * 2 + j) / a.G;
  // Scores stay unscaled up to the exponent, so their scale is made positive (a negative one's
  // sign goes to the queries) and 0 the least number above it, which keeps masked scores -inf.
  const float scale = a.scale_log2 == 0.f ? 1e-45f : fabsf(a.scale_log2);
  const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  auto start_segment = [&]() {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int r = rbase + n * 8 + g, rt = r / a.G;
      const T* q = reinterpret_cast<const T*>(a.q) + w.b * a.q_sb + rt * a.q_st +
                   (int64_t)(h * a.G + r - rt * a.G) * a.q_sh + c * 2;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[n][k][0] = (r < R ? *reinterpret_cast<const uint32_t*>(q + k * 16) : 0u) ^ sign;
        qf[n][k][1] = (r < R ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8) : 0u) ^ sign;
        o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[n][j] = -INFINITY;
        e[n][j] = l[n][j] = 0.f;
      }
    }
  };
  start_segment();

  // lane addresses of the ldmatrix tiles
  const uint32_t k_at = ((lane & 7) + ((lane >> 3) & 1) * 8) * PITCH + (lane >> 4) * 16;
  const uint32_t v_at = (TK + (lane & 7) + (lane >> 4) * 8) * PITCH + ((lane >> 3) & 1) * 16;
  int slot = 0;
  while (true) {
    cp_wait<ST - 2>();
    __syncwarp();
    issue(f);
    advance();
    const uint32_t tile = ring + slot * kStageBytes<D>;
    const unsigned char* vtile = ring_ptr + slot * kStageBytes<D> + TK * PITCH;
    slot = slot + 1 == ST ? 0 : slot + 1;
    float sc[MT][NB][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float s2[NB][4];   // one block: odd steps apart, two chains of dependent products
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[mt][n][j] = s2[n][j] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t kf[4];
        ldsm4(tile + k_at + mt * 16 * PITCH + k * 32, kf);
#pragma unroll
        for (int n = 0; n < NB; ++n) mma<DT>(NB == 1 && k & 1 ? s2[n] : sc[mt][n], kf, qf[n][k][0], qf[n][k][1]);
      }
      if constexpr (NB == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[mt][0][j] += s2[0][j];
      }
    }
    const Seq& s = w.s;
    const int key0 = (w.t < s.head ? w.t : w.t + s.jump) * TK;
    // a tile that every row sees whole needs no mask
    const int p_first = s.len - a.T;
    const bool open = key0 + TK <= p_first + 1 &&
                      (a.window == 0 || key0 + TK <= a.sinks || key0 > s.len - 1 - a.window);
    if (!open) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = key0 + mt * 16 + g + (j >> 1) * 8, p = p_first + tq[n][j & 1];
            const bool sees = key <= p && (a.window == 0 || key < a.sinks || key > p - a.window);
            if (!sees) sc[mt][n][j] = -INFINITY;
          }
    }
    // After the first tiles the maximum is rarely moved: one vote a tile then replaces the
    // reduction over the keys.
    float x[NB][2];
    bool past = false;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[n][j] = fmaxf(sc[0][n][j], sc[0][n][j + 2]);
#pragma unroll
        for (int mt = 1; mt < MT; ++mt) x[n][j] = fmaxf(x[n][j], fmaxf(sc[mt][n][j], sc[mt][n][j + 2]));
        x[n][j] *= scale;
        past |= x[n][j] > m[n][j] + (kLift + kSlack);
      }
    if (__any_sync(0xffffffffu, past)) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) x[n][j] = fmaxf(x[n][j], __shfl_xor_sync(0xffffffffu, x[n][j], w));
          const float to = fmaxf(m[n][j], x[n][j] - kLift);
          e[n][j] = to == -INFINITY ? 0.f : to;
          const float f2 = ex2(m[n][j] - e[n][j]);
          m[n][j] = to;
          l[n][j] *= f2;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            o[n][k][j] *= f2;
            o[n][k][j + 2] *= f2;
          }
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sc[mt][n][j] = ex2(fmaf(sc[mt][n][j], scale, -e[n][j & 1]));
          l[n][j & 1] += sc[mt][n][j];
        }
    // With several new tokens a masked key of this tile may be another row's
    // visible one, and 0 * (its infinity or NaN) would spoil this row: such a tile
    // is added element by element, masked keys left out. So is an infinity that is seen,
    // as a weight's two parts may meet it with opposite signs, or one of them be 0.
    bool odd = false;
    if ((!open && a.T > 1) || careful) {
      constexpr uint32_t EX = DT == DT_BF16 ? 0x7F80u : 0x7C00u;
      for (int id = lane; id < TK * CH; id += 32) {
        const uint4 u = *reinterpret_cast<const uint4*>(vtile + (id / CH) * PITCH + (id % CH) * 16);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= (w[j] & EX) == EX || ((w[j] >> 16) & EX) == EX;
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (!odd) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        // P has 11 bits in float16 and 8 in bfloat16; a second product adds what the
        // rounding left, which brings it to 22 and 16. (float16, 24 windowed sequences with four
        // drafts: without it 33.4 us and 39 % of the outputs rounded away from what float32
        // gives, a root mean square error of 3.75e-5; with it 35.1 us, 0.4 % and 3.28e-5.)
        uint32_t hi[NB][2], lo[NB][2];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float p0 = sc[mt][n][2 * u], p1 = sc[mt][n][2 * u + 1];
            hi[n][u] = pack2<DT>(p0, p1);
            const float2 back = unpack2<DT>(hi[n][u]);
            lo[n][u] = turn(pack2<DT>(p0 - back.x, p1 - back.y));
            hi[n][u] = turn(hi[n][u]);
          }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t vf[4];
          ldsm4t(tile + v_at + mt * 16 * PITCH + k * 32, vf);
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            mma<DT>(o[n][k], vf, hi[n][0], hi[n][1]);
            mma<DT>(o[n][k], vf, lo[n][0], lo[n][1]);
          }
        }
      }
    } else {
#pragma unroll 1
      for (int kk = 0; kk < TK; ++kk) {
        const int key = key0 + kk, from = (kk & 7) * 4 + c;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mine = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int u = 0; u < 2; ++u)
                if (kk / 8 == mt * 2 + u) mine = sc[mt][n][2 * u + j];
            const float w = __shfl_sync(0xffffffffu, mine, from);
            const int p = p_first + tq[n][j];
            if (!(key <= p && (a.window == 0 || key < a.sinks || key > p - a.window))) continue;
            const T* vrow = reinterpret_cast<const T*>(vtile + kk * PITCH);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              o[n][k][j] = fmaf(w, Elem<DT>::to_f(vrow[k * 16 + g]), o[n][k][j]);
              o[n][k][j + 2] = fmaf(w, Elem<DT>::to_f(vrow[k * 16 + g + 8]), o[n][k][j + 2]);
            }
          }
      }
    }
    const int was_b = w.b, was_t = w.t;
    const int64_t was_at = w.at;
    const bool whole_seq = seg0 == 0 && w.t + 1 == s.tiles;
    w.next(a, end);
    if (w.b != was_b || w.at >= end) {
      // the segment ends
      if (!careful) {
        // Looking for infinities tile by tile would cost every call; a sum that came out as no
        // number says that there are some, and the segment is taken again with the look.
        float all = 0.f;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int k = 0; k < KS; ++k) all += (o[n][k][0] + o[n][k][1]) + (o[n][k][2] + o[n][k][3]);
        if (__any_sync(0xffffffffu, all != all)) {
          careful = true;
          cp_wait<0>();
          __syncwarp();
          f.b = was_b;
          f.s = seq_of<TK>(a, was_b);
          f.t = seg0;
          f.at = was_at - (was_t - seg0);
          f.fetch(a, lane, whole);
          w = f;
          fill = 0;
          goto again;
        }
      }
      careful = false;
      // its sums over the lanes' keys, then out or to the workspace
      const bool done = whole_seq;
      const int64_t piece = ((int64_t)part * 2 + (started ? 0 : 1)) * cols + col;
      float2* ml = reinterpret_cast<float2*>(a.workspace) + piece * (8 * NB);
      float* po = reinterpret_cast<float*>(reinterpret_cast<float2*>(a.workspace) +
                                           (int64_t)parts * 2 * cols * (8 * NB)) + piece * (8 * NB) * D;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], w);
          const int lr = n * 8 + c * 2 + j, r = rbase + lr;
          if (r >= R) continue;
          const float sum = l[n][j];
          if (done) {
            const bool any = sum > 0.f || sum != sum;
            const float inv = any ? 1.f / sum : 0.f;
            const int64_t row = ((int64_t)was_b * a.T + tq[n][j]) * a.Hq + h * a.G + r - tq[n][j] * a.G;
            T* dst = reinterpret_cast<T*>(a.out) + row * D + g;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              dst[k * 16] = Elem<DT>::from_f(o[n][k][j] * inv);
              dst[k * 16 + 8] = Elem<DT>::from_f(o[n][k][j + 2] * inv);
            }
            if (a.lse != nullptr && g == 0) a.lse[row] = any ? m[n][j] * kLn2 + logf(sum) : -INFINITY;
          } else {
            if (g == 0) ml[lr] = make_float2(m[n][j], sum);
            float* dst = po + lr * D + g;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              dst[k * 16] = o[n][k][j];
              dst[k * 16 + 8] = o[n][k][j + 2];
            }
          }
        }
      if (w.at >= end) break;
      started = false;
      seg0 = 0;
      start_segment();
    }
  }
  cp_wait<0>();
}

// *p, or 0; in program order, so that many of them do not hold their addresses meanwhile.
__device__ __forceinline__ float load_if(const float* p, bool read) {
  float v;
  asm volatile(
      "{\n\t.reg .pred r;\n\tsetp.ne.s32 r, %2, 0;\n\tmov.f32 %0, 0f00000000;\n\t"
      "@r ld.global.f32 %0, [%1];\n\t}"
      : "=f"(v)
      : "l"(p), "r"((int)read)
      : "memory");
  return v;
}

// Joins the pieces of the sequences that were cut:
//   m = max m_i,  o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i,
// and fills the rows of empty sequences. A warp takes a row, or, for few rows of many
// pieces each (ROW_CTA), a CTA takes 32 dimensions of a row, a warp an eighth of the
// pieces.
// It fits beside the first kernel's CTAs, so it is launched and has its part boundaries
// when that one ends; but for four row blocks of head_dim 64, which fill the registers.
template <int DT, int D, bool ROW_CTA>
__global__ void __launch_bounds__(256, 4) decode_join_kernel(const DecodeArgs a, int parts) {
  constexpr int TK = Shape<D>::TK, NV = ROW_CTA ? 1 : D / 32, WARPS = 8, WPR = ROW_CTA ? WARPS : 1;
  __shared__ float red[WPR][34];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
  const int R = a.G * a.T, per = 8 * blocks_of(R, D), groups = row_groups(R, D), cols = a.Hkv * groups;
  const unsigned id = ROW_CTA ? blockIdx.x / (D / 32) : blockIdx.x * WARPS + warp;   // (b * Hkv + h) * R + r
  const int d0 = lane + (ROW_CTA ? (int)(blockIdx.x % (D / 32)) * 32 : 0);   // the lane's first dimension
  const unsigned head = id / (unsigned)R;
  const int r = (int)(id - head * R), b = (int)(head / (unsigned)a.Hkv), h = (int)(head - (unsigned)b * a.Hkv);
  if (b >= a.B) return;
  int64_t before, total;
  scan_to<TK>(a, lane, b, before, total);
  const int64_t chunk = max((int64_t)1, part_tiles(total, parts));
  const int n = seq_of<TK>(a, b).tiles;
  const int p0 = (int)quotient(before + kSeqCost, chunk);
  const int p1 = n > 0 ? (int)quotient(before + kSeqCost + n - 1, chunk) : p0;
  const bool late = before >= (int64_t)p0 * chunk;   // the sequence starts in its first part
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (n > 0 && p0 == p1) return;   // finished by its warp
  const int count = n > 0 ? p1 - p0 + 1 : 0;
  // the piece of part p0 + i, in slot 1 where the sequence starts
  const int64_t step = (int64_t)2 * cols * per, first = ((int64_t)p0 * 2 * cols + h * groups + r / per) * per + r % per;
  const int64_t zero = late ? (int64_t)cols * per : 0;
  const float2* ml = reinterpret_cast<const float2*>(a.workspace) + first;
  const float* po = reinterpret_cast<const float*>(reinterpret_cast<const float2*>(a.workspace) +
                                                   (int64_t)parts * step) + first * D + d0;
  // U pieces at a time, a lane the weight of one: their maxima, sums and outputs are all on
  // their way at once (with the maximum over all pieces taken first, 24 sequences of up to 17
  // pieces took 5.3 us here instead of 3.5, one of 148 pieces 6.0 instead of 2.8)
  constexpr int U = 24 / NV;
  float m = -INFINITY, acc[NV], l = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) acc[j] = 0.f;
  for (int i0 = sub; i0 < count; i0 += U * WPR) {
    const int mine = i0 + lane * WPR;
    float2 x = make_float2(-INFINITY, 0.f);
    if (lane < U && mine < count) x = ml[mine * step + (mine == 0 ? zero : 0)];
    float v[U][NV];
    const float* from = po + (i0 * step + (i0 == 0 ? zero : 0)) * D;
    const float* next = po + (i0 + WPR) * step * D;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NV; ++j) v[u][j] = load_if(from + 32 * j, i0 + u * WPR < count);
      from = next;
      next += WPR * step * D;
    }
    float to = fmaxf(m, x.x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, s));
    const float base = to == -INFINITY ? 0.f : to, f = ex2(m - base), w = ex2(x.x - base);
    m = to;
    l = fmaf(w, x.y, l * f);
#pragma unroll
    for (int j = 0; j < NV; ++j) acc[j] *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float wu = __shfl_sync(0xffffffffu, w, u);
#pragma unroll
      for (int j = 0; j < NV; ++j) acc[j] = fmaf(wu, v[u][j], acc[j]);
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
  if constexpr (ROW_CTA) {
    red[sub][lane] = acc[0];
    if (lane == 0) {
      red[sub][32] = l;
      red[sub][33] = m;
    }
    __syncthreads();
    if (sub != 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) m = fmaxf(m, red[w][33]);
    const float base = m == -INFINITY ? 0.f : m;
    acc[0] = l = 0.f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) {
      const float f = ex2(red[w][33] - base);
      acc[0] = fmaf(f, red[w][lane], acc[0]);
      l = fmaf(f, red[w][32], l);
    }
  }
  const bool any = l > 0.f || l != l;
  const float inv = any ? 1.f / l : 0.f;
  const int tq = r / a.G;
  const int64_t row = ((int64_t)b * a.T + tq) * a.Hq + h * a.G + r - tq * a.G;
  using E = Elem<DT>;
  typename E::T* dst = reinterpret_cast<typename E::T*>(a.out) + row * D;
#pragma unroll
  for (int j = 0; j < NV; ++j) dst[d0 + 32 * j] = E::from_f(acc[j] * inv);
  if (a.lse != nullptr && d0 == 0) a.lse[row] = any ? m * kLn2 + logf(l) : -INFINITY;
}

// Parts of the tile stream: with `cols` warps for each part, one wave of warps.
template <int D> int parts_for(int cols) {
  const int warps = kSms * Shape<D>::NW;
  return warps / cols > 0 ? warps / cols : 1;
}

template <int D> size_t workspace_for(int rows, int Hkv) {
  const int cols = Hkv * row_groups(rows, D);
  return (size_t)parts_for<D>(cols) * 2 * cols * 8 * blocks_of(rows, D) * (D + 2) * sizeof(float);
}


// A launch whose CTAs may come up while the kernel before it in the stream still runs;
// both kernels here wait for that one's end before they touch memory it may write.
template <typename... P>
cudaError_t launch_early(void (*kernel)(P...), int64_t blocks, int threads, int smem, cudaStream_t stream, P... p) {
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p...);
  if (e == cudaSuccess) count_launch();
  return e;
}

template <int DT, int D, int NB> cudaError_t launch_blocks(const DecodeArgs& a, cudaStream_t stream) {
  constexpr int NW = Shape<D>::NW, SMEM = NW * Shape<D>::ST * kStageBytes<D>;
  const int cols = a.Hkv * row_groups(a.G * a.T, D), parts = parts_for<D>(cols);
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_shared(reinterpret_cast<const void*>(decode_kernel<DT, D, NB>), SMEM, allowed);
  if (e != cudaSuccess) return e;
  e = launch_early(decode_kernel<DT, D, NB>, ((int64_t)parts * cols + NW - 1) / NW, NW * 32, SMEM, stream, a, parts);
  if (e != cudaSuccess) return e;
  const int64_t rows = (int64_t)a.B * a.Hq * a.T;
  // few rows with many pieces each: a CTA 32 dimensions of a row; else a warp a row
  return parts / a.B >= 16 ? launch_early(decode_join_kernel<DT, D, true>, rows * (D / 32), 256, 0, stream, a, parts)
                           : launch_early(decode_join_kernel<DT, D, false>, (rows + 7) / 8, 256, 0, stream, a, parts);
}

template <int DT, int D> cudaError_t launch_dim(const DecodeArgs& a, cudaStream_t stream) {
  const int blocks = blocks_of(a.G * a.T, D);
  if constexpr (D == 64)
    if (blocks == 4) return launch_blocks<DT, D, 4>(a, stream);
  return blocks == 1 ? launch_blocks<DT, D, 1>(a, stream) : launch_blocks<DT, D, 2>(a, stream);
}

template <int DT> cudaError_t launch_dt(const DecodeArgs& a, cudaStream_t stream) {
  switch (a.D) {
    case 64: return launch_dim<DT, 64>(a, stream);
    case 96: return launch_dim<DT, 96>(a, stream);
    case 128: return launch_dim<DT, 128>(a, stream);
    default: return launch_dim<DT, 256>(a, stream);
  }
}

}  // namespace

bool decode_supported(int D) { return D == 64 || D == 96 || D == 128 || D == 256; }

size_t decode_workspace_bytes(int T, int Hq, int Hkv, int D) {
  const int rows = Hq / Hkv * T;
  return D == 64 ? workspace_for<64>(rows, Hkv) : D == 96 ? workspace_for<96>(rows, Hkv)
       : D == 128 ? workspace_for<128>(rows, Hkv) : workspace_for<256>(rows, Hkv);
}

cudaError_t launch_decode(const DecodeArgs& a, int dt, cudaStream_t stream) {
  if (a.B == 0) return cudaSuccess;
  return dt == DT_BF16 ? launch_dt<DT_BF16>(a, stream) : launch_dt<DT_F16>(a, stream);
}

}  // namespace fpv2
