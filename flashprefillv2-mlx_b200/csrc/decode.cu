// Attention of the newest token (or the newest few) of every sequence over its
// paged K/V.
//
// Row t of sequence b sits at position p = len_b - T + t and sees key j when
// j <= p and (j < sinks or j > p - window); window 0 sees all j <= p.
//   o = sum_j softmax_j(scale q.k_j) v_j,   lse = log sum_j exp(scale q.k_j)
// A row that sees nothing gets o = 0 and lse = -inf.
//
// Every visible K and V row is read once for 4 G T D operations on 4 D bytes, so
// DRAM bandwidth bounds the call until G * T passes about 100 query rows; the
// tensor work is small and shaped 16 rows high, so it runs on mma.sync m16n8k16
// straight from shared memory, without TMEM round trips.
//
// Split: the visible keys of all sequences are one stream of TK-key tiles, cut
// into equal parts whatever the sequences' lengths are. One warp takes one part
// for one KV head (and one block of 16 query rows), with its own cp.async ring
// and running softmax, so warps never wait for each other; neighbouring warps
// take neighbouring heads of the same keys, which keeps the page reads of a
// block of threads contiguous. A sequence that lies inside one part is finished
// there; the pieces of the others go to the workspace in float32 and a second
// kernel, launched early and waiting for the first, joins them in part order, so
// the result does not depend on timing.
#include "common.cuh"
#include "kernels.h"

namespace fpv2 {
namespace {

constexpr int kSms = 148;      // B200; sets the split, so results do not vary with the device
constexpr float kLn2 = 0.6931471805599453f;

template <int D> struct Shape;   // keys a tile, ring stages, warps a CTA (about 200 KB of ring)
template <> struct Shape<64> { static constexpr int TK = 32, ST = 3, NW = 8; };
template <> struct Shape<96> { static constexpr int TK = 16, ST = 4, NW = 8; };
template <> struct Shape<128> { static constexpr int TK = 16, ST = 3, NW = 8; };
template <> struct Shape<256> { static constexpr int TK = 16, ST = 3, NW = 4; };

// Bytes between rows of a tile in shared memory: one 16-byte chunk more than the
// row, so the eight rows of an ldmatrix fall into different banks.
template <int D> constexpr int kPitch = D * 2 + 16;
template <int D> constexpr int kStageBytes = 2 * Shape<D>::TK * kPitch<D>;

__host__ __device__ inline int row_blocks(int G, int T) { return (G * T + 15) / 16; }

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

__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Tiles before sequence `want` and in total (warp-wide).
template <int TK>
__device__ __forceinline__ void scan_to(const DecodeArgs& a, int lane, int want, int64_t& before,
                                        int64_t& total) {
  before = total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int n = seq_of<TK>(a, b0 + lane).tiles;
    before += warp_sum(b0 + lane < want ? n : 0);
    total += warp_sum(n);
  }
}

__device__ __forceinline__ int64_t part_tiles(int64_t total, int parts) {
  return (total + parts - 1) / parts;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool read) {
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

// Walks the tiles of a part for the copies: sequence, tile in it, and the table
// entry of this lane's row, loaded one tile before it is needed.
template <int TK> struct Feed {
  int b, t;
  Seq s;
  int entry;

  __device__ __forceinline__ int key0() const { return (t < s.head ? t : t + s.jump) * TK; }
  __device__ __forceinline__ void fetch(const DecodeArgs& a, int lane) {
    const int key = min(key0() + lane % TK, s.len - 1);   // past the end: the last key's page
    entry = a.tables[(int64_t)b * a.table_stride + key / a.page_size];
  }
  __device__ __forceinline__ void next(const DecodeArgs& a, int lane, bool more) {
    if (!more) return;
    ++t;
    while (t >= s.tiles) {   // a part that goes on has a sequence with tiles ahead
      ++b;
      t = 0;
      s = seq_of<TK>(a, b);
    }
    fetch(a, lane);
  }
};

template <int DT, int D>
__global__ void __launch_bounds__(Shape<D>::NW * 32, 1) decode_kernel(const DecodeArgs a, int parts) {
  constexpr int TK = Shape<D>::TK, ST = Shape<D>::ST, NW = Shape<D>::NW;
  constexpr int PITCH = kPitch<D>, CH = D / 8, KS = D / 16, NT = TK / 8, ON = D / 8;
  using T = typename Elem<DT>::T;
  extern __shared__ __align__(16) unsigned char smem[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;   // mma fragment: rows g and g + 8, column pair c
  const int rbs = row_blocks(a.G, a.T), cols = a.Hkv * rbs;
  const int64_t wi = (int64_t)blockIdx.x * NW + warp;
  const int64_t part = wi / cols;
  const int col = (int)(wi - part * cols);
  const int h = col / rbs, rb = col - h * rbs;
  if (part >= parts) return;

  // this warp's range of the tile stream, and the sequence it starts in
  int64_t unused, total;
  scan_to<TK>(a, lane, 0, unused, total);
  const int64_t chunk = part_tiles(total, parts);
  const int64_t begin = part * chunk, end = min(begin + chunk, total);
  if (begin >= end) return;
  int count = (int)(end - begin);
  Feed<TK> f;
  {
    int64_t run = 0;
    int b0 = 0;
    while (true) {
      const int n = seq_of<TK>(a, b0 + lane).tiles;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, run + incl > begin);
      if (past) {
        const int at = __ffs(past) - 1;
        f.b = b0 + at;
        f.t = (int)(begin - run - (__shfl_sync(0xffffffffu, incl, at) - __shfl_sync(0xffffffffu, n, at)));
        break;
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
      b0 += 32;
    }
    f.s = seq_of<TK>(a, f.b);
  }
  f.fetch(a, lane);
  int b = f.b, t = f.t, seg0 = f.t;   // the consumer's sequence, tile, and the segment's first tile
  Seq s = f.s;
  bool first = true;

  const uint32_t ring = smem_u32(smem) + warp * ST * kStageBytes<D>;
  const T* kh = reinterpret_cast<const T*>(a.k) + h * a.k_sh;
  const T* vh = reinterpret_cast<const T*>(a.v) + h * a.v_sh;
  const bool whole_pages = a.page_size % TK == 0;
  int ahead = 0;   // tiles whose copies were issued

  auto issue = [&]() {
    if (ahead < count) {
      const uint32_t dst = ring + (ahead % ST) * kStageBytes<D>;
      const int key0 = f.key0();
      // element offsets of this lane's row (every lane of a whole page: row 0)
      const int page = clamp_entry(f.entry, 0, a.num_pages - 1, a.status);
      const int mine = whole_pages ? key0 : key0 + lane % TK;
      const int in_page = mine < f.s.len ? mine % a.page_size : 0;
      const int64_t ko = page * a.k_sp + in_page * a.k_sr, vo = page * a.v_sp + in_page * a.v_sr;
#pragma unroll
      for (int i = 0; i < TK * CH / 32; ++i) {
        const int id = lane + 32 * i, row = id / CH, ch = id % CH;
        int64_t kr = ko, vr = vo;
        if (whole_pages) {
          kr += row * a.k_sr;
          vr += row * a.v_sr;
        } else {
          kr = __shfl_sync(0xffffffffu, ko, row);
          vr = __shfl_sync(0xffffffffu, vo, row);
        }
        const int key = key0 + row;
        // keys that no row sees are zeros, whatever their page holds
        const bool seen = key < f.s.len && (key >= f.s.low || key < a.sinks);
        cp16(dst + row * PITCH + ch * 16, kh + kr + ch * 8, seen);
        cp16(dst + TK * PITCH + row * PITCH + ch * 16, vh + vr + ch * 8, seen);
      }
      ++ahead;
      f.next(a, lane, ahead < count);
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) issue();

  const int R = a.G * a.T;                       // query rows of a KV head
  const int r0 = rb * 16 + g, r1 = r0 + 8;       // this lane's two rows
  uint32_t qf[KS][4];
  float o[ON][4];
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  auto start_segment = [&]() {
    const int t0 = r0 / a.G, t1 = r1 / a.G;
    const T* q0 = reinterpret_cast<const T*>(a.q) + b * a.q_sb + t0 * a.q_st + (int64_t)(h * a.G + r0 - t0 * a.G) * a.q_sh;
    const T* q1 = reinterpret_cast<const T*>(a.q) + b * a.q_sb + t1 * a.q_st + (int64_t)(h * a.G + r1 - t1 * a.G) * a.q_sh;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int d = k * 16 + c * 2;
      qf[k][0] = r0 < R ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
      qf[k][1] = r1 < R ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
      qf[k][2] = r0 < R ? *reinterpret_cast<const uint32_t*>(q0 + d + 8) : 0u;
      qf[k][3] = r1 < R ? *reinterpret_cast<const uint32_t*>(q1 + d + 8) : 0u;
    }
#pragma unroll
    for (int n = 0; n < ON; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    m0 = m1 = -INFINITY;
    l0 = l1 = 0.f;
  };
  start_segment();

  for (int i = 0; i < count; ++i) {
    cp_wait<ST - 2>();
    __syncwarp();
    issue();
    const uint32_t kt = ring + (i % ST) * kStageBytes<D>, vt = kt + TK * PITCH;
    float sc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t kf[4];
        ldsm4(kt + (n * 8 + (lane & 7) + (lane >> 4) * 8) * PITCH + (2 * k + ((lane >> 3) & 1)) * 16, kf);
        mma<DT>(sc[n], qf[k], kf[0], kf[1]);
        mma<DT>(sc[n + 1], qf[k], kf[2], kf[3]);
      }
    }
    const int key0 = (t < s.head ? t : t + s.jump) * TK;
    // a tile that every row sees whole needs no mask
    const int p_first = s.len - a.T;
    const bool open = key0 + TK <= p_first + 1 && (a.window == 0 || key0 + TK <= a.sinks ||
                                                   key0 > s.len - 1 - a.window);
    const int p0 = p_first + r0 / a.G, p1 = p_first + r1 / a.G;
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v = sc[n][j] * a.scale_log2;
        if (!open) {
          const int key = key0 + n * 8 + c * 2 + (j & 1), p = j < 2 ? p0 : p1;
          const bool sees = key <= p && (a.window == 0 || key < a.sinks || key > p - a.window);
          v = sees ? v : -INFINITY;
        }
        sc[n][j] = v;
        if (j < 2)
          x0 = fmaxf(x0, v);
        else
          x1 = fmaxf(x1, v);
      }
    }
    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    const float e0 = n0 == -INFINITY ? 0.f : n0, e1 = n1 == -INFINITY ? 0.f : n1;
    if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
      const float a0 = ex2(m0 - e0), a1 = ex2(m1 - e1);
      l0 *= a0;
      l1 *= a1;
#pragma unroll
      for (int n = 0; n < ON; ++n) {
        o[n][0] *= a0;
        o[n][1] *= a0;
        o[n][2] *= a1;
        o[n][3] *= a1;
      }
      m0 = n0;
      m1 = n1;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      sc[n][0] = ex2(sc[n][0] - e0);
      sc[n][1] = ex2(sc[n][1] - e0);
      sc[n][2] = ex2(sc[n][2] - e1);
      sc[n][3] = ex2(sc[n][3] - e1);
      l0 += sc[n][0] + sc[n][1];
      l1 += sc[n][2] + sc[n][3];
    }
    // With several new tokens a masked key of this tile may be another row's
    // visible one, and 0 * (its infinity or NaN) would spoil this row: such a tile
    // is added element by element, masked keys left out.
    bool odd = false;
    if (!open && a.T > 1) {
      for (int id = lane; id < TK * CH; id += 32) {
        const uint4 u = *reinterpret_cast<const uint4*>(
            smem + (vt - smem_u32(smem)) + (id / CH) * PITCH + (id % CH) * 16);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        constexpr uint32_t EX = DT == DT_BF16 ? 0x7F80u : 0x7C00u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          odd |= (w[j] & EX) == EX || ((w[j] >> 16) & EX) == EX;
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (!odd) {
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        // P is held to 11 bits in float16; in bfloat16 (8 bits) a second product adds
        // what the rounding left, which brings it to 16.
        uint32_t pf[4] = {pack2<DT>(sc[n][0], sc[n][1]), pack2<DT>(sc[n][2], sc[n][3]),
                          pack2<DT>(sc[n + 1][0], sc[n + 1][1]), pack2<DT>(sc[n + 1][2], sc[n + 1][3])};
        uint32_t pl[4];
        if constexpr (DT == DT_BF16) {
          const float x[8] = {sc[n][0], sc[n][1], sc[n][2], sc[n][3],
                              sc[n + 1][0], sc[n + 1][1], sc[n + 1][2], sc[n + 1][3]};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 r = unpack2<DT>(pf[j]);
            pl[j] = pack2<DT>(x[2 * j] - r.x, x[2 * j + 1] - r.y);
          }
        }
#pragma unroll
        for (int d = 0; d < ON; d += 2) {
          uint32_t vf[4];
          ldsm4t(vt + (n * 8 + (lane & 7) + ((lane >> 3) & 1) * 8) * PITCH + (d + (lane >> 4)) * 16, vf);
          mma<DT>(o[d], pf, vf[0], vf[1]);
          mma<DT>(o[d + 1], pf, vf[2], vf[3]);
          if constexpr (DT == DT_BF16) {
            mma<DT>(o[d], pl, vf[0], vf[1]);
            mma<DT>(o[d + 1], pl, vf[2], vf[3]);
          }
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const int from = (lane & ~3) | (kk >> 1);
          const float w0 = __shfl_sync(0xffffffffu, sc[n][kk & 1], from);
          const float w1 = __shfl_sync(0xffffffffu, sc[n][2 + (kk & 1)], from);
          const int key = key0 + n * 8 + kk;
          const bool s0 = key <= p0 && (a.window == 0 || key < a.sinks || key > p0 - a.window);
          const bool s1 = key <= p1 && (a.window == 0 || key < a.sinks || key > p1 - a.window);
          const unsigned char* vrow = smem + (vt - smem_u32(smem)) + (n * 8 + kk) * PITCH;
#pragma unroll
          for (int d = 0; d < ON; ++d) {
            const float2 v = unpack2<DT>(*reinterpret_cast<const uint32_t*>(vrow + d * 16 + c * 4));
            if (s0) {
              o[d][0] = fmaf(w0, v.x, o[d][0]);
              o[d][1] = fmaf(w0, v.y, o[d][1]);
            }
            if (s1) {
              o[d][2] = fmaf(w1, v.x, o[d][2]);
              o[d][3] = fmaf(w1, v.y, o[d][3]);
            }
          }
        }
      }
    }
    ++t;
    if (t == s.tiles || i + 1 == count) {
      // the segment ends: its sums over the quad's columns, then out or to the workspace
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      if (seg0 == 0 && t == s.tiles) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int r = k ? r1 : r0;
          if (r >= R) continue;
          const float l = k ? l1 : l0, inv = l > 0.f || l != l ? 1.f / l : 0.f;
          const int tq = r / a.G;
          const int64_t row = ((int64_t)b * a.T + tq) * a.Hq + h * a.G + r - tq * a.G;
          T* dst = reinterpret_cast<T*>(a.out) + row * D + c * 2;
#pragma unroll
          for (int n = 0; n < ON; ++n)
            *reinterpret_cast<uint32_t*>(dst + n * 8) = pack2<DT>(o[n][2 * k] * inv, o[n][2 * k + 1] * inv);
          if (a.lse != nullptr && c == 0) a.lse[row] = l > 0.f || l != l ? (k ? m1 : m0) * kLn2 + logf(l) : -INFINITY;
        }
      } else {
        const int64_t slot = (part * 2 + (first ? 0 : 1)) * cols + col;
        float2* ml = reinterpret_cast<float2*>(a.workspace) + slot * 16;
        float* po = reinterpret_cast<float*>(reinterpret_cast<float2*>(a.workspace) + (int64_t)parts * 2 * cols * 16) +
                    slot * 16 * D;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int r = k ? r1 : r0, lr = g + 8 * k;
          if (r >= R) continue;
          if (c == 0) ml[lr] = k ? make_float2(m1, l1) : make_float2(m0, l0);
#pragma unroll
          for (int n = 0; n < ON; ++n)
            *reinterpret_cast<float2*>(po + lr * D + n * 8 + c * 2) = make_float2(o[n][2 * k], o[n][2 * k + 1]);
        }
      }
      first = false;
      if (i + 1 < count) {
        do {
          ++b;
          s = seq_of<TK>(a, b);
        } while (s.tiles == 0);
        t = 0;
        seg0 = 0;
        start_segment();
      }
    }
  }
  cp_wait<0>();
}

// Joins the pieces of the sequences that were cut:
//   m = max m_i,  o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i,
// and fills the rows of empty sequences. WPR warps take one query row.
template <int DT, int D, int WPR>
__global__ void __launch_bounds__(256) decode_join_kernel(const DecodeArgs a, int parts) {
  constexpr int TK = Shape<D>::TK, NV = D / 32;
  __shared__ float red[WPR > 1 ? WPR : 1][D + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR;
  const int64_t rows = (int64_t)a.B * a.T * a.Hq;
  const int64_t row_raw = (int64_t)blockIdx.x * (8 / WPR) + warp / WPR;
  const bool live = row_raw < rows;
  const int64_t row = live ? row_raw : rows - 1;
  const int hq = (int)(row % a.Hq), tq = (int)(row / a.Hq % a.T), b = (int)(row / a.Hq / a.T);
  const int h = hq / a.G, r = tq * a.G + hq - h * a.G;
  const int rbs = row_blocks(a.G, a.T), cols = a.Hkv * rbs, col = h * rbs + r / 16;
  int64_t before, total;
  scan_to<TK>(a, lane, b, before, total);
  const int64_t chunk = max((int64_t)1, part_tiles(total, parts));
  const int n = seq_of<TK>(a, b).tiles;
  const int64_t p0 = before / chunk, p1 = n > 0 ? (before + n - 1) / chunk : p0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n > 0 && p0 == p1) return;   // finished by its warp (the same for all warps of a row)
  const float2* ml = reinterpret_cast<const float2*>(a.workspace);
  const float* po = reinterpret_cast<const float*>(ml + (int64_t)parts * 2 * cols * 16);
  const int count = n > 0 ? (int)(p1 - p0 + 1) : 0;
  auto slot_row = [&](int i) {   // the piece of part p0 + i: a part's first segment is in its slot 0
    const int64_t p = p0 + i;
    const int64_t s = p * 2 + (i == 0 && before > p * chunk ? 1 : 0);
    return (s * cols + col) * 16 + r % 16;
  };
  float m = -INFINITY;
  for (int i = lane; i < count; i += 32) m = fmaxf(m, ml[slot_row(i)].x);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  const float base = m == -INFINITY ? 0.f : m;
  float acc[NV], l = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) acc[j] = 0.f;
#pragma unroll 4
  for (int i = sub; i < count; i += WPR) {
    const int64_t at = slot_row(i);
    const float2 x = ml[at];
    const float w = ex2(x.x - base);
    l = fmaf(w, x.y, l);
#pragma unroll
    for (int j = 0; j < NV; ++j) acc[j] = fmaf(w, po[at * D + lane + 32 * j], acc[j]);
  }
  if constexpr (WPR > 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) red[sub][lane + 32 * j] = acc[j];
    if (lane == 0) red[sub][D] = l;
    __syncthreads();
    if (sub != 0) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
#pragma unroll
      for (int j = 0; j < NV; ++j) acc[j] += red[w][lane + 32 * j];
      l += red[w][D];
    }
  }
  if (!live) return;
  const bool any = l > 0.f || l != l;
  const float inv = any ? 1.f / l : 0.f;
  using E = Elem<DT>;
  typename E::T* dst = reinterpret_cast<typename E::T*>(a.out) + row * D;
#pragma unroll
  for (int j = 0; j < NV; ++j) dst[lane + 32 * j] = E::from_f(acc[j] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[row] = any ? m * kLn2 + logf(l) : -INFINITY;
}

// Parts of the tile stream: with `cols` warps for each part, one wave of warps.
template <int D> int parts_for(int cols) {
  const int warps = kSms * Shape<D>::NW;
  return warps / cols > 0 ? warps / cols : 1;
}

template <int D> size_t workspace_for(int cols) {
  return (size_t)parts_for<D>(cols) * 2 * cols * 16 * (D + 2) * sizeof(float);
}

template <int DT, int D, int WPR>
cudaError_t launch_join(const DecodeArgs& a, int parts, cudaStream_t stream) {
  const int64_t rows = (int64_t)a.B * a.T * a.Hq;
  const int64_t blocks = (rows * WPR + 7) / 8;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, decode_join_kernel<DT, D, WPR>, a, parts);
  if (e == cudaSuccess) count_launch();
  return e;
}

template <int DT, int D> cudaError_t launch_dim(const DecodeArgs& a, cudaStream_t stream) {
  constexpr int NW = Shape<D>::NW, SMEM = NW * Shape<D>::ST * kStageBytes<D>;
  const int cols = a.Hkv * row_blocks(a.G, a.T), parts = parts_for<D>(cols);
  cudaError_t e = cudaFuncSetAttribute(decode_kernel<DT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e != cudaSuccess) return e;
  const int64_t blocks = ((int64_t)parts * cols + NW - 1) / NW;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  decode_kernel<DT, D><<<(unsigned)blocks, NW * 32, SMEM, stream>>>(a, parts);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  count_launch();
  // few rows with many pieces each: a CTA a row; else a warp a row
  return parts / a.B >= 16 ? launch_join<DT, D, 8>(a, parts, stream) : launch_join<DT, D, 1>(a, parts, stream);
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
  const int cols = Hkv * row_blocks(Hq / Hkv, T);
  return D == 64 ? workspace_for<64>(cols) : D == 96 ? workspace_for<96>(cols)
       : D == 128 ? workspace_for<128>(cols) : workspace_for<256>(cols);
}

cudaError_t launch_decode(const DecodeArgs& a, int dt, cudaStream_t stream) {
  if (a.B == 0) return cudaSuccess;
  return dt == DT_BF16 ? launch_dt<DT_BF16>(a, stream) : launch_dt<DT_F16>(a, stream);
}

}  // namespace fpv2
