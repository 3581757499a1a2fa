// Attention over the paged 8-bit KV cache (spatten_paged_attend).
//
// One pass over the cache. The R = H / G query heads of a KV head and the n
// new tokens of a sequence make n R query rows that share the keys; a row tile
// is 8 or 16 of them. Per 16 keys, on the tensor cores:
//   S^T [16 keys x 8 rows]  = K codes . q'^T,
//   O^T [D x 8 rows]       += V codes^T . P^T   (f16, every code is one; fp32 sums).
// A warp's tiles come through a ring of its own (cp.async, three tiles in
// flight; through registers the largest case below took 782 us). The order of the
// contracted dims (of S) and of the output dims (of O) is free, so each lane reads 16
// consecutive bytes of a row and takes them as fragments as they are, and every byte
// is read once per row tile. P^T turns from the layout of S^T into that of an operand
// with one 8x8 transpose (movmatrix).
//
// Bound by HBM where there are keys enough: 64 sequences x 8 heads x 32768 keys
// of int8, 660 to 680 us = 6.3 to 6.5 TB/s in short runs at full clocks; in a long run
// the GPU meets its power limit (990 W, 1.55 GHz instead of 1.97) and a call
// takes 676 to 726 us from one GPU to the next, 0.91 to 0.97 of the measured copy
// rate. One sequence of 131001, 53 us = 5.0 TB/s; 48 ragged ones of up to 8192, 79 us
// = 5.2 TB/s. One of 777 takes 8.8 us, which is the chain of dependent loads and the
// second launch. Beyond 16 rows each row tile walks the keys by itself: 32 sequences
// over 8192 keys of e4m3 take 100, 184, 274 and 379 us at 16, 32, 48 and 64 rows (the
// cache's bytes once: 82 us).
//
// Numerics:
//  * q' is the query row times a power of two, in what K's product takes: f16, or
//    an integer of three int8 terms beside int8 codes (Operands).
//  * s = (q' . codes) (sm_scale log2(e) k_scale / that power) in fp32, p =
//    2^(s - m) with a reference m that follows the row's maximum (updated when it is
//    exceeded by more than kSlack); l sums p in fp32.
//  * P is rounded to f16 for the second product (2^-11 of each weight, as much as
//    an fp16 output's own rounding: 2.7e-4 off the 64-bit result where fp32 weights
//    are 2.0e-4; a second f16 term would double that product), after v_scale has gone
//    into it: w = 2^(s + log2 v_scale - M), M a second reference
//    that follows max(s + log2 v_scale), kRoom below it. A block with a tiny scale and
//    all the weight keeps its 11 bits beside blocks with large scales and no weight,
//    and a weight down to 2^-21 of the row's largest beside that one (2^-32: half of
//    f16's smallest step).
//
// Work split, over one wave of resident CTAs and from the lengths on the device,
// so that a ragged batch and one long sequence fill the GPU alike and a captured
// launch follows the lengths it finds. A line is a (sequence, KV head, row tile).
// Few lines: each is cut into chunks of equal length, one per CTA (16 sequences x 8
// heads over up to 1000 keys: 22 -> 18 us). Many: the lines' units (16-key tiles,
// plus kLineCost for a line's set-up) are numbered and cut into equal ranges, one per
// CTA. The four warps of a CTA take turns on its tiles and join in shared memory; a
// (sequence, head, row tile) that a range's border cuts leaves (m, l, M, o) partials
// in the workspace, which a second kernel joins in a fixed order.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "kernels.h"
#include "paged_dev.cuh"
#include "paged_join.cuh"

namespace spatten {
namespace {

constexpr int kWarps = 4;
// What a line's set-up takes, in tiles (its chain of dependent loads and the
// join of the warps). Measured: 8 tiles are 7 % slower at 64 sequences of up to
// 2000 keys, 24 tiles 2 % at 48 of up to 8192.
constexpr uint32_t kLineCost = 16;
constexpr float kNone = -3.402823466e38f;  // reference of a row without a key: finite, so that -inf less it is -inf
constexpr uint32_t kNoRow = 0xFFFFFFFFu;
constexpr int kKeys = 16;  // of a tile, which lies within one page

// sequences whose prefix sums fit the shared memory
constexpr int kMaxBatch = 8192;

using Workspace = PagedPartials;

// What the products take. Every code of either type is an f16 (an int8's byte x ^
// 0x80 in the low byte of 0x6400 is the f16 1152 + x, and the difference is exact),
// and f16 queries keep what they have (query_scale).
//
// Beside int8 codes, one block of eight query rows has another form, in which the
// codes go into integer products as they are: three int8 terms a query, q' =
// 65536 q1 + 256 q2 + q3 rounded to an integer of at most 2^22, with exact sums.
// Without the widening of K, 64 sequences x 8 heads x 32768 keys take 666 us, bound
// by HBM alone; with it 697, and 818 instead of 734 on a GPU that its power limit
// slows down. The rounding is 2^-22 of the row's largest element, and within
// what a sum of D fp32 products is off by where that element is at most kOutlier
// times the row's mean magnitude; a tile with a row beyond takes the f16 form. (With
// two row blocks the widening is shared by 16 rows, and f16 is faster than two terms
// were: drafts of 24 sequences 22.0 -> 20.6 us.)
constexpr float kOutlier = 16.f;

template <int KV, int D, int NB>
struct Operands {
  static constexpr int KW = D / 16;  // K words of a lane and key
  static constexpr bool kTerms = KV == kKvInt8 && NB == 1;
  uint32_t q[NB][KW][kTerms ? 3 : 2];

  // f: the lane's dims of its query row, as the words hold them, times `up`
  SPATTEN_DEV void set(int nb, const float (&f)[KW][4], float up) {
#pragma unroll
    for (int w = 0; w < KW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h)  // in pairs as widen() brings them
        q[nb][w][h] = KV == kKvInt8 ? pack2<__half>(f[w][h] * up, f[w][2 + h] * up)
                                    : pack2<__half>(f[w][2 * h] * up, f[w][2 * h + 1] * up);
  }
  // the integer form: digits of f times kTermsUp `up`
  static constexpr float kTermsUp = 128.f;
  SPATTEN_DEV void set_terms(const float (&f)[KW][4], float up) {
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      uint32_t d[3] = {0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int x = __float2int_rn(f[w][i] * up * kTermsUp);
#pragma unroll
        for (int t = 2; t >= 0; --t) {
          const int low = (int)(int8_t)x;
          d[t] |= ((uint32_t)low & 0xFFu) << (8 * i);
          x = (x - low) >> 8;
        }
      }
#pragma unroll
      for (int t = 0; t < 3; ++t) q[0][w][t] = d[t];
    }
  }
  static SPATTEN_DEV uint32_t biased(uint32_t w) {
    const uint32_t u = (w & 0x00FF00FFu) ^ 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // a word's codes: int8's bytes (0, 2) and (1, 3), e4m3's (0, 1) and (2, 3)
  static SPATTEN_DEV void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (KV == kKvInt8) {
      lo = biased(w);
      hi = biased(w >> 8);
    } else {
      asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }"
          : "=r"(lo), "=r"(hi) : "r"(w));
    }
  }
  template <bool TERMS>
  SPATTEN_DEV void scores(const uint32_t (&k0)[KW], const uint32_t (&k1)[KW], float (&s)[NB][4]) const {
    if constexpr (TERMS) {
      int d[3][4];
#pragma unroll
      for (int t = 0; t < 3; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[t][i] = 0;
#pragma unroll
      for (int w = 0; w < KW; w += 2) {
        const uint32_t a[4] = {k0[w], k1[w], k0[w + 1], k1[w + 1]};
#pragma unroll
        for (int t = 0; t < 3; ++t) mma_s8_16832(d[t], a, q[0][w][t], q[0][w + 1][t]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[0][i] = fmaf((float)(256 * d[0][i] + d[1][i]), 256.f, (float)d[2][i]);
    } else {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[nb][i] = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        uint32_t a[4];
        widen(k0[w], a[0], a[2]);
        widen(k1[w], a[1], a[3]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma_16816<__half>(s[nb], a, q[nb][w][0], q[nb][w][1]);
      }
    }
  }
  // words of two keys: the key pairs of dims 0 .. 3
  static SPATTEN_DEV void values(uint32_t x, uint32_t y, uint32_t (&d)[4]) {
    if constexpr (KV == kKvInt8) {
      widen(__byte_perm(x, y, 0x5410), d[0], d[1]);
      widen(__byte_perm(x, y, 0x7632), d[2], d[3]);
    } else {
      widen(__byte_perm(x, y, 0x5140), d[0], d[1]);
      widen(__byte_perm(x, y, 0x7362), d[2], d[3]);
    }
  }
};

SPATTEN_DEV uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Row tiles of a sequence, and key tiles that its last row sees (one at least,
// so that rows without a key are written).
SPATTEN_DEV int row_tiles(const PagedSeq& s, int R, int rows) { return (int)(((int64_t)s.n * R + rows - 1) / rows); }
SPATTEN_DEV int key_tiles(const PagedSeq& s) { return max(1, (min(s.old + s.n, s.len) + kKeys - 1) / kKeys); }

template <int D, int NB>
struct Shape {
  static constexpr int kRows = 8 * NB;
  static constexpr int kStages = 4;              // tiles of a warp's ring
  static constexpr int kCtas = 3;                // resident per SM
  static constexpr int kBlockBytes = kKeys * D;  // K or V codes of a tile
  static constexpr int kStageBytes = 2 * kBlockBytes;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kOPad = D + 4;            // floats of a row in the join, which reuses the ring
  static_assert(kWarps * kRows * kOPad * 4 <= kRing, "the join fits the ring");
};

// 16-byte chunks of a block's rows, XOR-swizzled so that the fragment reads of
// eight lanes (two rows of K, or two chunks of four rows of V) meet different banks.
template <int D>
SPATTEN_DEV int swizzled(int row, int chunk) {
  if constexpr (D == 128) return row * 128 + ((chunk ^ (row & 7)) << 4);
  else return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}

// Offsets of a lane's pieces in a block of the ring: its rows' swizzles make two of
// each kind, the others are constant distances away.
template <int D>
struct LaneOffsets {
  uint32_t load[2], k[2], v[2];
  SPATTEN_DEV LaneOffsets(int lane) {
    constexpr int CH = D / 16;
    const int gid = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      load[i] = swizzled<D>(i * (32 / CH) + lane / CH, lane % CH) - i * 512;
      k[i] = swizzled<D>(gid, tig * (D / 64) + (D == 128 ? i : 0));
      v[i] = D == 128 ? swizzled<D>(2 * tig + i, gid) : swizzled<D>(2 * tig + i, gid >> 1) + (gid & 1) * 8;
    }
  }
};

// A block of 16 rows into the ring; rows at or behind `live` arrive as zeros
// (their bytes may be anything).
template <int D>
SPATTEN_DEV void load_block(uint32_t dst, const LaneOffsets<D>& lo, const uint8_t* src, int lane, int live) {
  constexpr int CH = D / 16, RPI = 32 / CH;  // chunks per row, rows per warp instruction
#pragma unroll
  for (int i = 0; i < 16 / RPI; ++i) {
    const int row = i * RPI + lane / CH;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst + lo.load[i & 1] + i * 512),
                 "l"(src + i * 512), "r"(row < live ? 16 : 0));
  }
}

SPATTEN_DEV uint4 lds128(uint32_t a) {
  uint4 x;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(a));
  return x;
}
SPATTEN_DEV uint2 lds64(uint32_t a) {
  uint2 x;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(a));
  return x;
}

// Words of K row gid + 8 h for lane tig: dims (D / 4) tig .. + D / 4 - 1.
template <int D>
SPATTEN_DEV void read_k(uint32_t (&k)[D / 16], uint32_t blk, const LaneOffsets<D>& lo, int h) {
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const uint4 x = lds128(blk + lo.k[j] + 8 * h * D);
    k[4 * j] = x.x; k[4 * j + 1] = x.y; k[4 * j + 2] = x.z; k[4 * j + 3] = x.w;
  }
}

// Words of V row 2 tig + (r & 1) + 8 (r >> 1) for lane gid: dims (D / 8) gid .. + D / 8 - 1.
template <int D>
SPATTEN_DEV void read_v(uint32_t (&v)[D / 32], uint32_t blk, const LaneOffsets<D>& lo, int r) {
  const uint32_t at = blk + lo.v[r & 1] + 8 * (r >> 1) * D;
  if constexpr (D == 128) {
    const uint4 x = lds128(at);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
    const uint2 x = lds64(at);
    v[0] = x.x; v[1] = x.y;
  }
}

template <int KV, int D, int NB>
__global__ void __launch_bounds__(32 * kWarps, Shape<D, NB>::kCtas)
paged_attend_kernel(const PagedAttendParams p, const Workspace ws, const bool bf16) {
  using SH = Shape<D, NB>;
  using Ops = Operands<KV, D, NB>;
  constexpr int ROWS = SH::kRows, KS = D / 16, NT = 32 * kWarps;
  constexpr int AHEAD = 32;  // tiles whose pages and scales a warp holds
  constexpr int ST = SH::kStages;
  extern __shared__ __align__(128) uint8_t dsm[];
  float (*sm_o)[ROWS][SH::kOPad] = reinterpret_cast<float (*)[ROWS][SH::kOPad]>(dsm);  // over the rings
  uint32_t* pre = reinterpret_cast<uint32_t*>(dsm + SH::kRing);  // [B + 1] units before each sequence
  __shared__ float sm_m[kWarps][ROWS], sm_l[kWarps][ROWS], sm_M[kWarps][ROWS];
  __shared__ uint32_t scan[2 * kWarps];
  __shared__ unsigned long long scan_most[kWarps];
  grid_dependents();
  grid_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
  const int G = p.c.G, R = p.b.H / G, page = p.c.page, page_log = __ffs(page) - 1;
  const LaneOffsets<D> offs(lane);
  const uint8_t* const k_lane = p.c.k + lane * 16;
  const uint8_t* const v_lane = p.c.v + lane * 16;

  // tiles and lines in all. The host made sure of 32 bits for sequences
  // that share no rows; others may need more, and then nothing is done.
  unsigned long long most = 0;
  uint32_t U = 0, lines = 0;
  auto tiles_of = [&](int b, uint32_t& n) {  // key tiles of a line of sequence b, and its lines
    n = 0;
    if (b >= p.b.B) return 0u;
    const PagedSeq s = paged_seq(p.b, p.c, b);
    if (paged_serves(p, s, R)) n = (uint32_t)G * row_tiles(s, R, ROWS);
    return (uint32_t)key_tiles(s);
  };
  uint32_t n0, k0 = 0;  // of sequence `tid`
  for (int base = 0; base < p.b.B; base += NT) {
    uint32_t n;
    const uint32_t k = tiles_of(base + tid, n);
    if (base == 0) {
      n0 = n;
      k0 = k;
    }
    const uint32_t x = __reduce_add_sync(0xffffffffu, n * k), y = __reduce_add_sync(0xffffffffu, n);
    unsigned long long z = (unsigned long long)n * (k + kLineCost);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) {
      scan[warp] = x;
      scan[kWarps + warp] = y;
      scan_most[warp] = z;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      U += scan[w];
      lines += scan[kWarps + w];
      most += scan_most[w];
    }
    __syncthreads();
  }
  if (most >> 32) U = lines = 0;
  // chunk: tiles per unit. ceil(tiles / chunk) summed over the lines is at most
  // U / chunk + lines, so with few lines every unit has a CTA.
  // It takes U lines / (grid (grid - lines)) tiles more than an equal share, and
  // saves most CTAs a line's set-up.
  const bool few = lines * 2 <= gridDim.x &&
                   (float)U * lines <= (float)kLineCost * gridDim.x * (gridDim.x - lines);
  const uint32_t chunk = few ? max((U + gridDim.x - lines - 1) / (gridDim.x - lines), (uint32_t)kWarps) : 1;
  const uint32_t lead = few ? 0 : kLineCost;
  auto units_of = [&](uint32_t k) { return few ? (k + chunk - 1) / chunk : k + lead; };
  // prefix sums of the sequences' units
  U = 0;
  if (tid == 0) pre[0] = 0;
  for (int base = 0; base < p.b.B; base += NT) {
    uint32_t n = n0, k = k0;
    if (base > 0) k = tiles_of(base + tid, n);
    uint32_t x = n * units_of(k);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    uint32_t before = U;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      U += scan[w];
    }
    if (base + tid < p.b.B) pre[base + tid + 1] = before + x;
    __syncthreads();
  }
  if (most >> 32) U = 0;
  const uint32_t cta = blockIdx.x;
  const uint32_t ctas = min(gridDim.x, few ? U : (U + kWarps - 1) / kWarps);
  PagedCut cut = {};
  if (cta >= ctas) {
    if (tid == 0) ws.cut[cta] = cut;
    return;
  }
  const uint32_t per = U / ctas, more = U % ctas;  // the first `more` CTAs take one unit more
  uint32_t u = cta * per + min(cta, more);
  const uint32_t u1 = u + per + (cta < more ? 1 : 0);
  int b = 0;
  for (int hi = p.b.B; hi - b > 1;) {  // the sequence of unit u
    const int mid = (b + hi) >> 1;
    if (pre[mid] <= u) b = mid; else hi = mid;
  }

  while (u < u1) {
    while (pre[b + 1] <= u) ++b;
    const PagedSeq sq = paged_seq(p.b, p.c, b);
    const uint32_t KT = key_tiles(sq), KU = units_of(KT), RT = row_tiles(sq, R, ROWS);
    const uint32_t local = u - pre[b], line = local / KU, v0 = local % KU, v1 = min(KU, v0 + (u1 - u));
    const int g = line / RT, rt = line % RT;
    const uint32_t t0 = few ? v0 * chunk : max(v0, lead) - lead, t1 = few ? min(KT, v1 * chunk) : max(v1, lead) - lead;
    const int nrows = sq.n * R, r0 = rt * ROWS;
    // slots that the tile's last and first row see
    const int lim_max = min(sq.old + min((r0 + ROWS - 1) / R, sq.n - 1) + 1, sq.len);
    const int lim_min = min(sq.old + r0 / R + 1, sq.len);
    const uint32_t t_end = min(t1, (uint32_t)(max(lim_max, 0) + kKeys - 1) / kKeys);

    // queries: row gid of each 8-row block, all dims of it in the four lanes of gid
    uint4 raw[NB][KS / 2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = r0 + nb * 8 + gid;
      const uint16_t* qp = static_cast<const uint16_t*>(p.q) + (D / 4) * tig;
      if (r < nrows) qp += (int64_t)(sq.begin + r / R) * p.q_st + (int64_t)(g * R + r % R) * p.q_sh;
#pragma unroll
      for (int s = 0; s < KS / 2; ++s)
        raw[nb][s] = r < nrows ? *(reinterpret_cast<const uint4*>(qp) + s) : make_uint4(0u, 0u, 0u, 0u);
    }

    // this warp's tiles t0 + warp, + 4, ..: lane i keeps the row offset and the
    // scales of tile i of the AHEAD tiles at hand, and the page of the one AHEAD
    // tiles on
    const int nt = t_end > t0 + warp ? (t_end - t0 - warp + kWarps - 1) / kWarps : 0;
    auto tile_slot = [&](int j) { return (int)(t0 + warp + kWarps * j) * kKeys; };
    auto page_of = [&](int j) {
      const int slot = tile_slot(j + lane);
      return slot < lim_max ? paged_page(p.c, b, slot >> page_log) : -1;
    };
    auto row_of = [&](int j, int pid) {
      const int slot = tile_slot(j + lane);
      return pid >= 0 ? ((uint32_t)pid * G + g) * page + (slot & (page - 1)) : kNoRow;
    };
    const uint32_t ring = smem_u32(dsm) + warp * ST * SH::kStageBytes;
    uint32_t row_l = kNoRow, have_l = 0, have_n = 0;  // have: tiles with memory, a bit per lane
    int pid_n = -1;
    float ks_l = 0.f, vs_l = 0.f, ks_n = 0.f, vs_n = 0.f;
    // tile j on its way into slot j % ST (an empty group past the end)
    auto issue = [&](int j) {
      if (j < nt) {
        const int at = j % AHEAD;
        if (at == 0) {
          const int pid = j == 0 ? page_of(0) : pid_n;
          row_l = row_of(j, pid);
          have_n = __ballot_sync(0xffffffffu, pid >= 0);
          const int64_t blk = (int64_t)max(pid, 0) * G + g;
          ks_n = pid >= 0 ? *(p.c.k_scale + blk) : 0.f;
          vs_n = pid >= 0 ? *(p.c.v_scale + blk) : 0.f;
          if (nt > j + AHEAD) pid_n = page_of(j + AHEAD);
        }
        const uint32_t dst = ring + (j % ST) * SH::kStageBytes;
        const uint32_t row = __shfl_sync(0xffffffffu, row_l, at);
        const uint64_t off = row == kNoRow ? 0 : (uint64_t)row * D;
        load_block<D>(dst, offs, k_lane + off, lane, row == kNoRow ? 0 : kKeys);
        load_block<D>(dst + SH::kBlockBytes, offs, v_lane + off, lane, row == kNoRow ? 0 : lim_max - tile_slot(j));
      }
      cp_async_commit();
    };
#pragma unroll
    for (int j = 0; j < ST - 1; ++j) issue(j);

    Ops ops;
    float cq[NB][2], m[NB][2], M[NB][2], l[NB][2];
    int lim[NB][2];
    float o[NB][KS][4];
    bool terms = false;  // the integer form of the scores
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float f[KS][4], top = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 four = raw[nb][s / 2];
          const uint32_t w = s & 1 ? (j ? four.w : four.z) : (j ? four.y : four.x);
          float2 x;
          if (bf16) x = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
          else x = __half22float2(*reinterpret_cast<const __half2*>(&w));
          f[s][2 * j] = x.x;
          f[s][2 * j + 1] = x.y;
          top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
          // fmaxf drops a NaN: it makes the row's factor NaN instead
          if (!(x.x == x.x && x.y == x.y)) top = INFINITY;
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      QueryScale qs = query_scale(top, p.scale_log2);
      if constexpr (Ops::kTerms) {
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum += fabsf(f[s][j]);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        terms = __all_sync(0xffffffffu, !(top > kOutlier / D * sum));  // (rows that are not finite: either)
      }
      if (terms) {
        if constexpr (Ops::kTerms) ops.set_terms(f, qs.up);
        qs.factor *= 1.f / Ops::kTermsUp;
      } else {
        ops.set(nb, f, qs.up);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // this lane's rows of the products: 2 tig, 2 tig + 1
        cq[nb][j] = __shfl_sync(0xffffffffu, qs.factor, (2 * tig + j) * 4);
        lim[nb][j] = min(sq.old + (r0 + nb * 8 + 2 * tig + j) / R + 1, sq.len);
        m[nb][j] = M[nb][j] = kNone;
        l[nb][j] = 0.f;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[nb][s][j] = 0.f;
    }

    auto tiles = [&](auto form) {
      constexpr bool TERMS = decltype(form)::value;
      for (int j = 0; j < nt; ++j) {
        cp_async_wait<ST - 2>();
        __syncwarp();  // tile j has landed for every lane, and tile j - 1 is read
        issue(j + ST - 1);
        const uint32_t stage = ring + (j % ST) * SH::kStageBytes;
        const int slot0 = tile_slot(j), at = j % AHEAD;
        if (at == 0) {
          have_l = have_n;
          ks_l = ks_n;
          vs_l = vs_n > 0.f ? fmaxf(log2f(vs_n), kNoScale) : kNoScale;  // log2 of the scale
        }
        const float ks = __shfl_sync(0xffffffffu, ks_l, at), lv = __shfl_sync(0xffffffffu, vs_l, at);
        const bool none = !((have_l >> at) & 1u);
        float s[NB][4];
        uint32_t k0[KS], k1[KS];
        read_k<D>(k0, stage, offs, 0);
        read_k<D>(k1, stage, offs, 1);
        ops.template scores<TERMS>(k0, k1, s);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float f0 = cq[nb][0] * ks, f1 = cq[nb][1] * ks;
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nb][i] *= i & 1 ? f1 : f0;
        }
        if (slot0 + kKeys > lim_min || none) {  // warp-uniform
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (none || slot0 + gid + 4 * (i & 2) >= lim[nb][i & 1]) s[nb][i] = -INFINITY;
        }
        // p = 2^(s - m), and w = 2^(s + log2 v_scale - M)
        float top[NB][2], topw[NB][2];  // largest s, and s + log2 v_scale, of this lane
        bool up = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            top[nb][c] = fmaxf(s[nb][c], s[nb][2 + c]);
            topw[nb][c] = top[nb][c] + lv;
            up |= top[nb][c] > m[nb][c] + kSlack || topw[nb][c] > M[nb][c] + (kRoom + kSlack);
          }
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = top[nb][c], y = topw[nb][c];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) {
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
              }
              const float mn = fmaxf(m[nb][c], x), Mn = fmaxf(M[nb][c], y - kRoom);
              l[nb][c] *= fast_exp2(m[nb][c] - mn);
              const float f = fast_exp2(M[nb][c] - Mn);
#pragma unroll
              for (int k = 0; k < KS; ++k) {
                o[nb][k][c] *= f;
                o[nb][k][2 + c] *= f;
              }
              m[nb][c] = mn;
              M[nb][c] = Mn;
            }
        }
        uint32_t pf[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float m0 = m[nb][0], m1 = m[nb][1], M0 = M[nb][0], M1 = M[nb][1];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float s0 = s[nb][2 * i], s1 = s[nb][2 * i + 1];
            l[nb][0] += fast_exp2(s0 - m0);
            l[nb][1] += fast_exp2(s1 - m1);
            pf[nb][i] = transpose8x8(pack2<__half>(fast_exp2(s0 + (lv - M0)), fast_exp2(s1 + (lv - M1))));
          }
        }
        // values
        uint32_t v[4][D / 32];
#pragma unroll
        for (int r = 0; r < 4; ++r) read_v<D>(v[r], stage + SH::kBlockBytes, offs, r);
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          uint32_t lo[4], hi[4];
          Ops::values(v[0][w], v[1][w], lo);
          Ops::values(v[2][w], v[3][w], hi);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a[4] = {lo[2 * h], lo[2 * h + 1], hi[2 * h], hi[2 * h + 1]};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma_16816<__half>(o[nb][2 * w + h], a, pf[nb][0], pf[nb][1]);
          }
        }
      }
    };
    if constexpr (Ops::kTerms) {
      if (terms) tiles(std::true_type{}); else tiles(std::false_type{});
    } else {
      tiles(std::false_type{});
    }
    __syncthreads();  // every ring is read

    // the warps join, sums by m and outputs by M
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = nb * 8 + 2 * tig + c;
        float sum = l[nb][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        float4* dst = reinterpret_cast<float4*>(&sm_o[warp][row][gid * (D / 8)]);
#pragma unroll
        for (int k = 0; k < KS; k += 2)
          dst[k / 2] = make_float4(o[nb][k][c], o[nb][k][2 + c], o[nb][k + 1][c], o[nb][k + 1][2 + c]);
        if (gid == 0) {
          sm_m[warp][row] = m[nb][c] == kNone ? -INFINITY : m[nb][c];
          sm_l[warp][row] = sum;
          sm_M[warp][row] = M[nb][c] == kNone ? -INFINITY : M[nb][c];
        }
      }
    __syncthreads();
    const bool whole = v0 == 0 && v1 == KU;
    const int slot = 2 * cta + (v0 == 0 ? 1 : 0);
    for (int i = tid; i < ROWS * (D / 4); i += NT) {
      const int row = i / (D / 4), d = (i % (D / 4)) * 4, r = r0 + row;
      if (r >= nrows) break;
      float mm = -INFINITY, MM = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        mm = fmaxf(mm, sm_m[w][row]);
        MM = fmaxf(MM, sm_M[w][row]);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = fast_exp2(sm_M[w][row] - finite_or_0(MM));
        const float4 x = *reinterpret_cast<const float4*>(&sm_o[w][row][d]);
        ll += sm_l[w][row] * fast_exp2(sm_m[w][row] - finite_or_0(mm));
        acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
      }
      if (whole) {
        const float inv = paged_normaliser(mm, ll, MM);
        uint16_t* op = static_cast<uint16_t*>(p.out) + (int64_t)(sq.begin + r / R) * p.o_st +
                       (int64_t)(g * R + r % R) * p.o_sh + d;
        uint2 v;
        v.x = bf16 ? pack2<__nv_bfloat16>(acc.x * inv, acc.y * inv) : pack2<__half>(acc.x * inv, acc.y * inv);
        v.y = bf16 ? pack2<__nv_bfloat16>(acc.z * inv, acc.w * inv) : pack2<__half>(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(op) = v;
      } else {
        *reinterpret_cast<float4*>(ws.o + ((int64_t)slot * ROWS + row) * D + d) = acc;
        if (d == 0) ws.ml[(int64_t)slot * ROWS + row] = make_float4(mm, ll, MM, 0.f);
      }
    }
    if (v0 == 0 && !whole) {  // cut: the CTAs up to that of its last unit hold a part each
      const uint32_t last = u + KU - 1, big = more * (per + 1);
      cut.parts = (int)(last < big ? last / (per + 1) : more + (last - big) / per) - (int)cta + 1;
      cut.row0 = r0; cut.nrows = nrows; cut.begin = sq.begin; cut.g = g;
    }
    __syncthreads();
    u += v1 - v0;
  }
  if (tid == 0) ws.cut[cta] = cut;
}

// Eight query rows per pass where that covers a sequence's rows (the register
// tile of 16 has room for half the bytes in flight), else sixteen.
int row_block(const PagedAttendParams& p) {
  // beside the tcgen05 launch: what is left is mostly single tokens
  const int64_t tokens = p.rows_upto <= kTcRows ? 1 : p.b.max_tokens;
  return tokens * (p.b.H / p.c.G) <= 8 ? 8 : 16;
}

double units_bound(const PagedAttendParams& p) {
  const int rows = row_block(p);
  const double lines = (double)p.b.T * (p.b.H / p.c.G) / rows + p.b.B;  // row tiles of all sequences, at most
  return lines * p.c.G * ((double)p.c.max_pages * p.c.page / 16 + 1 + kLineCost);
}

// One resident wave, and no more than could have a unit for each warp.
int grid_ctas(const PagedAttendParams& p, int n_sm) {
  const int wave = n_sm * 3;
  return (int)fmin((double)wave, fmax(1.0, ceil(units_bound(p) / kWarps)));
}

template <int KV, int D, int NB>
cudaError_t attend_launch(const PagedAttendParams& p, bool bf16, const Workspace& ws, int ctas, cudaStream_t st) {
  using SH = Shape<D, NB>;
  const size_t smem = SH::kRing + (size_t)(p.b.B + 1) * sizeof(uint32_t);
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may use its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
    e = cudaFuncSetAttribute(paged_attend_kernel<KV, D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             SH::kRing + (kMaxBatch + 1) * (int)sizeof(uint32_t));
    if (e != cudaSuccess) return e;
    if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  e = launch_dependent(paged_attend_kernel<KV, D, NB>, dim3(ctas), 32 * kWarps, smem, st, p, ws, bf16);
  if (e != cudaSuccess) return e;
  return launch_paged_join<D, SH::kRows>(p, ws, ctas, bf16, st);
}

template <int KV, int D>
cudaError_t attend_rows(const PagedAttendParams& p, bool bf16, const Workspace& ws, int ctas, cudaStream_t st) {
  return row_block(p) == 8 ? attend_launch<KV, D, 1>(p, bf16, ws, ctas, st)
                           : attend_launch<KV, D, 2>(p, bf16, ws, ctas, st);
}

template <int KV>
cudaError_t attend_dim(const PagedAttendParams& p, bool bf16, const Workspace& ws, int ctas, cudaStream_t st) {
  if (p.c.D == 128) return attend_rows<KV, 128>(p, bf16, ws, ctas, st);
  if (p.c.D == 64) return attend_rows<KV, 64>(p, bf16, ws, ctas, st);
  return cudaErrorInvalidValue;
}

}  // namespace

int paged_attend_max_batch() { return kMaxBatch; }

namespace {

// Which kernels a call takes. Sequences of more than kTcRows query rows per KV
// head (pieces of prompts) go to the tcgen05 kernel, the others to the one above.
// 64 rows (8 KV heads x 128, int8) take 40 us there and 43 us here at 4 sequences
// over 4096 keys, 61 and 71 us at one over 32768, 349 and 476 us at 32 over 8192, but
// 49 and 44 us at 16 over 1000 (e4m3) and 24 and 15 us at one over 800; 96 rows 40
// and 57, 60 and 94, 331 and 702, 50 and 56, 24 and 15 us. So the sides meet at 40
// rows where sequences are many and long and beyond 128 where they are few and short;
// the border is in between, as lengths are not known on the host, which
// knows the largest sequence's rows only. Where
// the rows show that some must be shorter, both are launched and each serves its
// own, so that single tokens beside a prompt's piece keep the kernel made for
// them (512 new tokens over 4096 take 63 us, 47 single ones over 4000 76, together
// 150).
struct Plan {
  PagedAttendParams tc, few;
  bool use_tc, use_few;
};

Plan plan_for(const PagedAttendParams& p) {
  Plan x = {p, p, false, true};
  x.tc.rows_over = x.few.rows_over = 0;
  x.tc.rows_upto = x.few.rows_upto = INT64_MAX;
  if (!paged_attend_tc_takes(p)) return x;
  x.use_tc = true;
  x.use_few = p.b.B > 1 && p.b.T < (int64_t)p.b.B * p.b.max_tokens;
  if (x.use_few) x.tc.rows_over = x.few.rows_upto = kTcRows;
  return x;
}

}  // namespace

bool paged_attend_fits(const PagedAttendParams& p) { return units_bound(plan_for(p).few) < 4e9; }

size_t paged_attend_workspace(const PagedAttendParams& p, int n_sm) {
  const Plan x = plan_for(p);
  return (x.use_tc ? paged_attend_tc_workspace(p, n_sm) : 0) +
         (x.use_few ? paged_partials_bytes(grid_ctas(x.few, n_sm), row_block(x.few), p.c.D) : 0);
}

cudaError_t launch_paged_attend(const PagedAttendParams& p, int dtype, int kv, void* ws, int n_sm, cudaStream_t st) {
  if (dtype != kF16 && dtype != kBF16) return cudaErrorInvalidValue;
  const Plan x = plan_for(p);
  uint8_t* w = static_cast<uint8_t*>(ws);
  if (x.use_tc) {
    const cudaError_t e = launch_paged_attend_tc(x.tc, dtype, kv, w, n_sm, st);
    if (e != cudaSuccess || !x.use_few) return e;
    w += paged_attend_tc_workspace(p, n_sm);
  }
  const int ctas = grid_ctas(x.few, n_sm);
  const Workspace s = paged_partials(w, ctas, row_block(x.few));
  const bool bf16 = dtype == kBF16;
  return kv == kKvInt8 ? attend_dim<kKvInt8>(x.few, bf16, s, ctas, st) : attend_dim<kKvE4m3>(x.few, bf16, s, ctas, st);
}

}  // namespace spatten
