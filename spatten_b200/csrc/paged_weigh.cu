// The weights that the new tokens give the cached ones (spatten_paged_attend_ext
// with weights): after the attention, whose statistics (m, 1 / l) of each row are
// read,
//   weight[slot] = (slot is an earlier token's ? weight[slot] : 0) + sum over rows
//                  of 2^(q . k sm_scale log2(e) - m) / l
// for every slot that a row of the call may see; the new tokens' slots take their
// positions. Two ways, by the query rows that a sequence has per KV head:
//
// Up to kScoreRows: the attention has kept its scores (4 bytes a row and slot), and
// paged_weigh_scores_kernel (paged_weigh_rowed_kernel beyond 8 rows) turns them into weights.
// For 64 sequences x 8 heads x 32768
// keys with 4 rows the scores and weights are 670 MB to write and read; reading the keys
// again would take 2.1 GB (2806 us with a kernel that did, 830 to 880 now, the attention alone
// 665 to 690; the scores' kernel by itself 64 us = 5.5 TB/s, what is left is the
// attention's stores and the second launch). One user's step over 777 keys: 12.2 us
// of device time, 9.0 without weights.
//
// More: the scores are computed again, on the tensor cores, with the keys as rows:
//   S^T [128 keys x 128 rows] = K codes . Q'^T   (kind::f16, fp32 in tensor memory),
// so that a thread owns a key and the sum over rows needs no exchange.
// paged_weigh_rows_kernel lays the query rows out once (f16 as the attention's, in
// the layout that the MMAs read, and two numbers a row: cq, its scores' factor, and
// b = log2(1 / l) - m, so that p = 2^(S (cq k_scale) + b), cq mostly the same for a
// tile); paged_weigh_tc_kernel
// takes 256 keys x a chunk of the rows at a time; the last kernel adds the chunks up.
// Bound by the exponentials, one per (row, key): 1024 new tokens over 8192, 2 sequences, 16
// / 8 heads, e4m3: 92 us for 185 million of them, 64 % of the conversion pipe's cycles
// while an SM has work, tensor pipe 33 %; 259 us with the attention, which takes 152.
// What it took: the keys widened a block ahead by warps of their own (four warps that sum per
// scheduler instead of two CTAs that do everything by turns), and code that fits the
// instruction caches: the same kernel with its rare paths unrolled took 145 us.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "kernels.h"
#include "paged_dev.cuh"
#include "sm100.cuh"

namespace spatten {
namespace {

using namespace sm100;

// ---------------------------------------------------------------- slots

// The kernels that write weights: a thread takes four slots (of one page), so that it
// has 16 bytes of their weights in each access, and a CTA a group of heads.
constexpr int kSlotThreads = 256, kQuad = 4, kSlotsCta = kSlotThreads * kQuad;

struct WeighSlots {
  int slot, lim;  // the first one; the sequence's end
  int old;        // slots from here on are new tokens'
  int64_t row;    // of head 0

  // false: no memory, or behind the end
  SPATTEN_DEV bool set(const PagedWeighParams& p, const PagedSeq& sq, int b, int first) {
    const PagedCache& c = p.a.c;
    slot = first;
    lim = min(sq.old + sq.n, sq.len);
    old = sq.old;
    if (slot >= lim) return false;
    const int pid = paged_page(c, b, slot / c.page);
    row = (int64_t)max(pid, 0) * c.G * c.page + slot % c.page;
    return pid >= 0;
  }
  SPATTEN_DEV bool plain() const { return slot + kQuad <= min(lim, old); }  // earlier tokens' all
  // A head's weights before the call (their bytes; finish() knows which count).
  SPATTEN_DEV float4 before(const PagedWeighParams& p, int g) const {
    return *reinterpret_cast<const float4*>(p.weight + row + (int64_t)g * p.a.c.page);
  }
  SPATTEN_DEV void finish(const PagedWeighParams& p, const PagedSeq& sq, int g, float4 was, const float (&add)[kQuad]) const {
    const int64_t at = row + (int64_t)g * p.a.c.page;
    if (plain()) {
      *reinterpret_cast<float4*>(p.weight + at) = make_float4(was.x + add[0], was.y + add[1], was.z + add[2], was.w + add[3]);
      return;
    }
    const float w[kQuad] = {was.x, was.y, was.z, was.w};
#pragma unroll
    for (int i = 0; i < kQuad; ++i) {
      if (slot + i >= lim) break;
      const bool fresh = slot + i >= old;
      p.weight[at + i] = (fresh ? 0.f : w[i]) + add[i];
      if (fresh) p.position[at + i] = p.positions ? p.positions[sq.begin + slot + i - old] : slot + i;
    }
  }
};

// Where what is kept for a slot lies: of head 0, and from a head to the next.
struct SlotPlaces {
  int64_t first, head;
  SPATTEN_DEV SlotPlaces(const PagedAttendParams& a, int b, int slot, int64_t row) {
    const int64_t slots = (int64_t)a.c.max_pages * a.c.page;
    first = a.by_pool ? row : (int64_t)b * a.c.G * slots + slot;
    head = a.by_pool ? a.c.page : slots;
  }
};

// Slots x sequences x groups of heads; groups of `heads`, smaller where the CTAs are few.
dim3 slot_grid(const PagedWeighParams& p, int n_sm, int per_cta, int& heads) {
  const int64_t slots = (int64_t)p.a.c.max_pages * p.a.c.page, G = p.a.c.G;
  const int64_t ctas = (slots + per_cta - 1) / per_cta;
  heads = 8;
  while (heads > 1 && ctas * p.a.b.B * ((G + heads - 1) / heads) < 4 * n_sm) heads /= 2;
  return dim3((unsigned)ctas, p.a.b.B, (unsigned)((G + heads - 1) / heads));
}

// ---------------------------------------------------------------- few rows: kept scores

template <int ROWS>
__global__ void __launch_bounds__(kSlotThreads) paged_weigh_scores_kernel(const PagedWeighParams p, int heads) {
  __shared__ float2 stat[8][ROWS];
  grid_dependents();
  grid_wait();
  const PagedAttendParams& a = p.a;
  const int b = blockIdx.y, G = a.c.G, R = a.b.H / G, g0 = blockIdx.z * heads, tid = threadIdx.x;
  const PagedSeq sq = paged_seq(a.b, a.c, b);
  const int nrows = sq.n * R;
  if (sq.n == 0 || nrows > p.rows_over) return;
  WeighSlots x;
  const bool live = x.set(p, sq, b, blockIdx.x * kSlotsCta + kQuad * tid);
  static_assert(8 * ROWS <= kSlotThreads, "a row's statistics per thread");
  if (tid < heads * ROWS && g0 + tid / ROWS < G) {
    const int g = g0 + tid / ROWS, r = tid % ROWS;
    if (r < nrows) stat[tid / ROWS][r] = a.stat[(int64_t)(sq.begin + r / R) * a.b.H + g * R + r % R];
  }
  __syncthreads();
  if (!live) return;
  const SlotPlaces place(a, b, x.slot, x.row);
  const float* src = a.score + place.first * ROWS;
#pragma unroll 2
  for (int h = 0; h < min(heads, G - g0); ++h) {
    const int g = g0 + h;
    const float4* at = reinterpret_cast<const float4*>(src + g * place.head * ROWS);
    const float4 was = x.before(p, g);
    float add[kQuad] = {0.f, 0.f, 0.f, 0.f};
    float s[kQuad * ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const float4 y = __ldcs(at + i);  // (read once)
      s[4 * i] = y.x; s[4 * i + 1] = y.y; s[4 * i + 2] = y.z; s[4 * i + 3] = y.w;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < nrows) {
        const float2 y = stat[h][r];
#pragma unroll
        for (int i = 0; i < kQuad; ++i) add[i] += fast_exp2(s[i * ROWS + r] - y.x) * y.y;
      }
    x.finish(p, sq, g, was, add);
  }
}

// 16 or 32 rows a slot: four rows a thread, so that a slot's scores are read whole (four
// slots a thread as above: 50 us for the 42 at 24 sequences of 7 drafted tokens over 2000).
constexpr int kRowedSlots = 64;  // of a CTA

template <int ROWS>
__global__ void __launch_bounds__(kSlotThreads) paged_weigh_rowed_kernel(const PagedWeighParams p, int heads) {
  constexpr int L = ROWS / 4, SPP = kSlotThreads / L;  // threads of a slot, slots of a pass
  __shared__ float2 stat[8][ROWS];
  grid_dependents();
  grid_wait();
  const PagedAttendParams& a = p.a;
  const int b = blockIdx.y, G = a.c.G, R = a.b.H / G, g0 = blockIdx.z * heads, tid = threadIdx.x, li = tid % L;
  const PagedSeq sq = paged_seq(a.b, a.c, b);
  const int nrows = sq.n * R, first = blockIdx.x * kRowedSlots, lim = min(sq.old + sq.n, sq.len);
  if (sq.n == 0 || nrows > p.rows_over || first >= lim) return;  // (the CTA as one)
  static_assert(8 * ROWS <= kSlotThreads, "a row's statistics per thread");
  if (tid < heads * ROWS && g0 + tid / ROWS < G) {
    const int g = g0 + tid / ROWS, r = tid % ROWS;
    stat[tid / ROWS][r] = r < nrows ? a.stat[(int64_t)(sq.begin + r / R) * a.b.H + g * R + r % R] : make_float2(0.f, 0.f);
  }
  __syncthreads();
  // the attention's tiles of rows store each up to the last slot that one of them sees
  int sees[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) sees[k] = 4 * li + k >= nrows ? 0 : a.tree ? INT_MAX : sq.old + (4 * li + k) / R + 1;
  // (little code, which runs a few times, and many warps)
#pragma unroll 1
  for (int s0 = 0; s0 < kRowedSlots; s0 += SPP) {
    const int slot = first + s0 + tid / L;
    const int pid = slot < lim ? paged_page(a.c, b, slot / a.c.page) : -1;
    const int64_t row = (int64_t)max(pid, 0) * G * a.c.page + slot % a.c.page;
    const SlotPlaces place(a, b, slot, row);
#pragma unroll 1
    for (int h = 0; h < min(heads, G - g0); ++h) {
      const int g = g0 + h;
      const int64_t at = row + (int64_t)g * a.c.page;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      if (pid >= 0 && 4 * li < nrows)
        y = __ldcs(reinterpret_cast<const float4*>(a.score + (place.first + g * place.head) * ROWS) + li);
      const float before = pid >= 0 && li == 0 && slot < sq.old ? p.weight[at] : 0.f;
      const float s[4] = {y.x, y.y, y.z, y.w};
      float add = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 z = stat[h][4 * li + k];
        if (slot < sees[k]) add += fast_exp2(s[k] - z.x) * z.y;
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
      if (pid >= 0 && li == 0) {
        p.weight[at] = before + add;
        if (slot >= sq.old) p.position[at] = p.positions ? p.positions[sq.begin + slot - sq.old] : slot;
      }
    }
  }
}

cudaError_t scores_launch(const PagedWeighParams& p, int n_sm, cudaStream_t st) {
  int heads;
  const dim3 grid = slot_grid(p, n_sm, p.a.score_rows > 8 ? kRowedSlots : kSlotsCta, heads);
  switch (p.a.score_rows) {
    case 1: return launch_dependent(paged_weigh_scores_kernel<1>, grid, kSlotThreads, 0, st, p, heads);
    case 2: return launch_dependent(paged_weigh_scores_kernel<2>, grid, kSlotThreads, 0, st, p, heads);
    case 4: return launch_dependent(paged_weigh_scores_kernel<4>, grid, kSlotThreads, 0, st, p, heads);
    case 8: return launch_dependent(paged_weigh_scores_kernel<8>, grid, kSlotThreads, 0, st, p, heads);
    case 16: return launch_dependent(paged_weigh_rowed_kernel<16>, grid, kSlotThreads, 0, st, p, heads);
    case 32: return launch_dependent(paged_weigh_rowed_kernel<32>, grid, kSlotThreads, 0, st, p, heads);
    default: return cudaErrorInvalidValue;
  }
}

// ---------------------------------------------------------------- many rows: tensor cores

constexpr int kKeys = 256, kTileRows = 128, kGroup = 32, kFoldTiles = 4;
constexpr int kSumWarps = 16, kWideWarps = 4, kThreads = 32 * (kSumWarps + kWideWarps + 2);
constexpr int kRing = 2;    // tiles of query rows, blocks of keys in shared memory
constexpr int kConsts = 4;  // tiles' row constants
constexpr int kConstBytes = kTileRows * 8 + 16;  // b and cq of the rows, the cq that all have (0: each its own)
constexpr unsigned kErr = 0x500;
constexpr uint32_t kNoRow = 0xFFFFFFFFu;

// What the main kernel works on, in the workspace.
struct WeighPlan {
  uint8_t* tiles;     // [G][tiles_g] records: 128 query rows, then their constants
  float* partial;     // [chunks][2][places]: sums of the even and the odd 64 rows of a chunk's tiles
  int64_t places;     // slot_places
  int64_t tiles_g;
  int chunk, chunks;  // rows of a chunk (a multiple of kTileRows), chunks of a sequence at most
};

template <int D>
struct Lay {
  static constexpr int kQBytes = kTileRows * D * 2;
  static constexpr int kRecord = kQBytes + kConstBytes;
  static constexpr int kKHalf = 128 * D * 2;
  static constexpr int oK = 0;                               // [ring][2][D / 64][128][128 B]
  static constexpr int oQ = oK + kRing * 2 * kKHalf;         // [ring][D / 64][128][128 B]
  static constexpr int oC = oQ + kRing * kQBytes;            // [kConsts]
  static constexpr int oScale = oC + kConsts * kConstBytes;  // [ring][256] scales of the keys
  static constexpr int oRow = oScale + kRing * kKeys * 4;    // [ring][256] rows of the pool
  static constexpr int oItem = oRow + kRing * kKeys * 4;     // [ring] Item
  static constexpr int oBar = oItem + kRing * 64;
  static constexpr int kBars = 4 * kRing + 2 * kConsts + 4 + 1;
  static constexpr int oTmem = oBar + kBars * 8;
  static constexpr int oAbort = oTmem + 4;
  static constexpr int oScan = (oAbort + 4 + 7) & ~7;        // [warps] 64-bit
  static constexpr int oPre = oScan + 8 * (kThreads / 32);   // [pairs + 1]
  static constexpr int bytes(int B) { return oPre + ((B + 1) / 2 + 1) * 4 + 1024; }
};

constexpr int kRowThreads = 512;

// First record of sequence b: records of sequences whose rows are apart are apart.
SPATTEN_DEV int64_t first_tile(const PagedSeq& s, int R, int b) { return (int64_t)s.begin * R / kTileRows + b; }

template <int D>
__global__ void __launch_bounds__(kRowThreads) paged_weigh_rows_kernel(const PagedWeighParams p, const WeighPlan w, bool bf16) {
  using L = Lay<D>;
  constexpr int LQ = D / 8, RPP = kRowThreads / LQ;  // lanes of a row, rows of a pass
  grid_dependents();
  grid_wait();
  const PagedAttendParams& a = p.a;
  // whose record this is (a CTA for each of the longest sequence's tiles in every sequence would be
  // half a million where one prompt of 8192 tokens is among 256 sequences)
  __shared__ int owner;
  const int g = blockIdx.y, R = a.b.H / a.c.G, tid = threadIdx.x;
  if (tid == 0) owner = -1;
  __syncthreads();
  for (int i = tid; i < a.b.B; i += kRowThreads) {
    const PagedSeq s = paged_seq(a.b, a.c, i);
    const int64_t at = (int64_t)blockIdx.x - first_tile(s, R, i);
    if (s.n * R > p.rows_over && at >= 0 && at * kTileRows < s.n * R) atomicMax(&owner, i);
  }
  __syncthreads();
  const int b = owner;
  if (b < 0) return;
  const PagedSeq sq = paged_seq(a.b, a.c, b);
  const int nrows = sq.n * R, t = (int)(blockIdx.x - first_tile(sq, R, b));
  uint8_t* rec = w.tiles + (g * w.tiles_g + blockIdx.x) * (int64_t)L::kRecord;
  const int li = tid % LQ;
  auto pair = [&](uint32_t x) {
    return bf16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u))
                : __half22float2(*reinterpret_cast<const __half2*>(&x));
  };
  constexpr int STEPS = kTileRows / RPP;
  uint4 x[STEPS];
  float top[STEPS], most = 0.f;  // the rows' largest magnitudes, that of the finite rows of the tile
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int r = t * kTileRows + k * RPP + tid / LQ;
    x[k] = make_uint4(0u, 0u, 0u, 0u);
    if (r < nrows)
      x[k] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (int64_t)(sq.begin + r / R) * a.q_st +
                                             (int64_t)(g * R + r % R) * a.q_sh + 8 * li);
  }
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const uint32_t in[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = pair(in[j]);
      m = fmaxf(m, fmaxf(fabsf(f.x), fabsf(f.y)));
      if (!(f.x == f.x && f.y == f.y)) m = INFINITY;  // fmaxf drops a NaN
    }
#pragma unroll
    for (int d = LQ / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    top[k] = m;
    if (m < INFINITY) most = fmaxf(most, m);
  }
  __shared__ float red[kRowThreads / 32];
  most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
  if ((tid & 31) == 0) red[tid >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 32; ++i) most = fmaxf(most, red[i]);
  // One power of two for the tile, so that the sums need one number a row instead of two: where
  // each row reaches 2^-12 of the largest magnitude, which goes to 2^14 or more, its own largest is 4
  // or more: what f16 drops of it, at most half its smallest step 2^-24, is below 2^-27 of that.
  bool far = false;
#pragma unroll
  for (int k = 0; k < STEPS; ++k) far |= top[k] > 0.f && top[k] < most * 0x1p-12f;
  const bool common = !__syncthreads_or(far);
  float* const consts = reinterpret_cast<float*>(rec + L::kQBytes);
  const QueryScale all = query_scale(most, a.scale_log2);
  if (tid == 0) consts[2 * kTileRows] = common ? all.factor : 0.f;
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int y = k * RPP + tid / LQ, r = t * kTileRows + y;
    const uint32_t in[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
    const QueryScale own = query_scale(top[k], a.scale_log2);  // (its factor is NaN for a row that is not finite)
    const float up = top[k] < INFINITY ? (common ? all.up : own.up) : 0.f;
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = pair(in[j]);
      o[j] = up > 0.f ? pack2<__half>(f.x * up, f.y * up) : 0u;
    }
    *reinterpret_cast<uint4*>(rec + (li >> 3) * (kTileRows * 128) + y * 128 + (((li & 7) ^ (y & 7)) << 4)) =
        make_uint4(o[0], o[1], o[2], o[3]);
    if (li == 0) {
      float2 c = make_float2(-INFINITY, 0.f);  // no row: no weight
      if (r < nrows) {
        const float2 s = a.stat[(int64_t)(sq.begin + r / R) * a.b.H + g * R + r % R];
        c = make_float2(top[k] < INFINITY ? log2f(s.y) - s.x : NAN, common ? all.factor : own.factor);
      }
      consts[y] = c.x;
      consts[kTileRows + y] = c.y;
    }
  }
}

SPATTEN_DEV void bulk_load(uint32_t dst, const void* src, uint32_t bytes, SBar bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar.a)
               : "memory");
}

// Waits for the loads under way; r, which one of them fills, is used behind this only.
SPATTEN_DEV void tmem_wait_ld32(float (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
               "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
               "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
               "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
               ::"memory");
}

// Four codes in order as two f16 pairs.
template <int KV>
SPATTEN_DEV uint2 widen4(uint32_t w) {
  if constexpr (KV == kKvInt8) {
    const uint32_t x = w ^ 0x80808080u;  // byte u under 0x64 is the f16 1024 + u = 1152 + code
    uint32_t lo = __byte_perm(x, 0x64646464u, 0x4140), hi = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 b = __half2half2(__ushort_as_half(0x6480));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&lo), b);
    const __half2 z = __hsub2(*reinterpret_cast<const __half2*>(&hi), b);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&y), *reinterpret_cast<const uint32_t*>(&z));
  } else {
    return make_uint2(e4m3x2_to_f16x2(w & 0xFFFFu), e4m3x2_to_f16x2(w >> 16));
  }
}

// What the sums and the products have to know of a block of keys. The warps that widen
// it leave it beside it: working it out took each of the others a quarter of an item's time.
struct Item {
  int t0, t1;            // row tiles; none: the last item is behind
  int k0, lim;           // first slot, end of the sequence
  int old, n, begin;     // of its PagedSeq
  int nrows;
  int64_t partial;       // where the even rows' sums go, of the first slot or of row 0 of the pool
};
static_assert(sizeof(Item) <= 64, "two of them in Lay");

// The items of a CTA: 256 keys of a (sequence, KV head) by a chunk of its rows.
struct Items {
  const PagedWeighParams& p;
  const WeighPlan& w;
  const uint32_t* pre;  // items before each pair of sequences
  int R;
  uint32_t next_item, total;
  // the sequence: its items, its blocks of keys and chunks of rows
  uint32_t from, to, kt, ch;
  PagedSeq sq;
  int b, lim, nrows;
  // the item: row tiles [t0, t1)
  int g, c, k0, t0, t1;

  static SPATTEN_DEV int limit(const PagedSeq& s) { return max(min(s.old + s.n, s.len), 0); }
  static SPATTEN_DEV unsigned long long count(const PagedWeighParams& p, const WeighPlan& w, int b) {
    if (b >= p.a.b.B) return 0;
    const PagedSeq s = paged_seq(p.a.b, p.a.c, b);
    const int R = p.a.b.H / p.a.c.G, rows = s.n * R;
    if (rows <= p.rows_over) return 0;
    return (unsigned long long)p.a.c.G * ((rows + w.chunk - 1) / w.chunk) * ((limit(s) + kKeys - 1) / kKeys);
  }
  SPATTEN_DEV Items(const PagedWeighParams& p, const WeighPlan& w, const uint32_t* pre, uint32_t first, uint32_t total)
      : p(p), w(w), pre(pre), R(p.a.b.H / p.a.c.G), next_item(first), total(total), from(0), to(0) {}
  SPATTEN_DEV bool next() {
    while (next_item < total) {
      const uint32_t u = next_item;
      next_item += gridDim.x;
      if (u < from || u >= to) {
        int lo = 0;
        for (int hi = (p.a.b.B + 1) / 2; hi - lo > 1;) {  // the pair of item u
          const int mid = (lo + hi) >> 1;
          if (pre[mid] <= u) lo = mid; else hi = mid;
        }
        b = 2 * lo;
        from = pre[lo];
        to = from + (uint32_t)count(p, w, b);
        if (u >= to) {
          ++b;
          from = to;
          to = pre[lo + 1];
        }
        sq = paged_seq(p.a.b, p.a.c, b);
        lim = limit(sq);
        nrows = sq.n * R;
        kt = (lim + kKeys - 1) / kKeys;
        ch = (nrows + w.chunk - 1) / w.chunk;
      }
      const uint32_t x = (u - from) / kt;
      k0 = (int)(u - from - x * kt) * kKeys;
      g = (int)(x / ch);
      c = (int)(x - g * ch);
      t0 = c * (w.chunk / kTileRows);
      t1 = min(t0 + w.chunk / kTileRows, (nrows + kTileRows - 1) / kTileRows);
      if (!p.a.tree && k0 > sq.old) t0 = max(t0, (int)min((int64_t)(k0 - sq.old) * R / kTileRows, (int64_t)INT_MAX));
      if (t0 < t1) return true;
    }
    return false;
  }
};

template <int KV, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_weigh_tc_kernel(const PagedWeighParams p, const WeighPlan w) {
  using L = Lay<D>;
  extern __shared__ uint8_t smem_raw[];
  grid_dependents();
  grid_wait();
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t bars = smem_u32(sm + L::oBar);
  const SBarArr q_full{bars}, q_empty{bars + 8 * kRing}, k_full{bars + 16 * kRing}, k_empty{bars + 24 * kRing},
      c_full{bars + 32 * kRing}, c_empty{bars + 32 * kRing + 8 * kConsts}, s_full{bars + 32 * kRing + 16 * kConsts},
      s_empty{bars + 32 * kRing + 16 * kConsts + 16}, rest{bars + 32 * kRing + 16 * kConsts + 32};
  const SBar drain = rest[0];
  volatile int* abort = reinterpret_cast<volatile int*>(sm + L::oAbort);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + L::oTmem);
  uint32_t* pre = reinterpret_cast<uint32_t*>(sm + L::oPre);
  unsigned long long* scan = reinterpret_cast<unsigned long long*>(sm + L::oScan);
  const PagedAttendParams& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.c.G, R = a.b.H / G;

  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(q_full[i], 1);
      mbar_init(q_empty[i], 1);
      mbar_init(k_full[i], kWideWarps);
      mbar_init(k_empty[i], kSumWarps + 1);  // the scales are read, and the products done
    }
    for (int i = 0; i < kConsts; ++i) {
      mbar_init(c_full[i], 1);
      mbar_init(c_empty[i], kSumWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full[i], 1);
      mbar_init(s_empty[i], kSumWarps);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
    *abort = 0;
    pre[0] = 0;
  }
  if (warp == kSumWarps + kWideWarps + 1) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  unsigned long long U = 0;
  const int pairs = (a.b.B + 1) / 2;
  for (int base = 0; base < pairs; base += kThreads) {
    const int i = base + tid;
    unsigned long long x = i < pairs ? Items::count(p, w, 2 * i) + Items::count(p, w, 2 * i + 1) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    unsigned long long front = U;
    for (int k = 0; k < kThreads / 32; ++k) {
      if (k < warp) front += scan[k];
      U += scan[k];
    }
    if (i < pairs) pre[i + 1] = (uint32_t)(front + x);
    __syncthreads();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  // (the attention's host check leaves 32 bits for sequences that share no rows)
  Items it(p, w, pre, blockIdx.x, U >> 32 ? 0u : (uint32_t)U);

  if (warp < kSumWarps) {
    // ------------------------------------------------------------ sums of the weights
    // a thread takes a key and half of a tile's rows (four warps per scheduler hide one
    // another's latencies, which two did not)
    constexpr int kHalf = kTileRows / 2;
    const int side = warp >> 3, key = tid & (kKeys - 1);
    const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + ((warp >> 2) & 1) * kTileRows + side * kHalf;
    uint32_t n = 0, items = 0;  // tiles, blocks of keys
    bool alive = true;
    while (alive) {
      const uint32_t kb = items % kRing;
      if (!__all_sync(0xffffffffu, mbar_wait(k_full[kb], (items / kRing) & 1, kErr | 8, abort))) break;
      const Item it = *reinterpret_cast<const Item*>(sm + L::oItem + kb * 64);
      if (it.t0 == it.t1) break;
      const float ks = *reinterpret_cast<const float*>(sm + L::oScale + (kb * kKeys + key) * 4);
      const uint32_t row = *reinterpret_cast<const uint32_t*>(sm + L::oRow + (kb * kKeys + key) * 4);
      __syncwarp();
      mbar_arrive_elect(k_empty[kb]);
      ++items;
      const int slot = it.k0 + key;
      float total = 0.f;
      float2 sum = make_float2(0.f, 0.f);
      const int last = min(it.k0 + (key | 31), it.lim - 1);  // key of the warp
      for (int t = it.t0; t < it.t1; ++t, ++n) {
        const uint32_t buf = n & 1, cs = n % kConsts;
        bool ok = mbar_wait(s_full[buf], (n >> 1) & 1, kErr | 1, abort);
        ok = ok && mbar_wait(c_full[cs], (n / kConsts) & 1, kErr | 2, abort);
        if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        tc_fence_after();
        const int r0 = t * kTileRows + side * kHalf, groups = (min(kHalf, it.nrows - r0) + kGroup - 1) / kGroup;
        // whether every row of the half sees the warp's keys: row r0 sees slots up to sq.old + r0 / R
        const bool seen = last < it.old || (!a.tree && (int64_t)(last - it.old) * R <= r0);
        // the first row of the half that sees the key, in the causal form
        const int f = a.tree || seen ? 0
                          : (int)min(max((int64_t)(slot - it.old) * R - r0, (int64_t)0), (int64_t)kHalf);
        const bool some = groups > 0 && __any_sync(0xffffffffu, f < kHalf);
        const float* cst = reinterpret_cast<const float*>(sm + L::oC + cs * kConstBytes);
        const float4* bs = reinterpret_cast<const float4*>(cst + side * kHalf);
        const float cq = cst[2 * kTileRows];
        const float2 f2 = make_float2(cq * ks, cq * ks);
        // (loops that are not unrolled keep the roles' code within the instruction caches)
        if (some && seen && cq != 0.f) {
#pragma unroll 1
          for (int q = 0; q < groups; ++q) {
            float s[kGroup];
            tmem_ld32f(ts + buf * 2 * kTileRows + q * kGroup, s);
            tmem_wait_ld32(s);
#pragma unroll
            for (int k = 0; k < kGroup / 4; ++k) {
              const float4 b = bs[q * (kGroup / 4) + k];
              float2 y = __ffma2_rn(make_float2(s[4 * k], s[4 * k + 1]), f2, make_float2(b.x, b.y));
              float2 z = __ffma2_rn(make_float2(s[4 * k + 2], s[4 * k + 3]), f2, make_float2(b.z, b.w));
              y = make_float2(fast_exp2(y.x), fast_exp2(y.y));
              z = make_float2(fast_exp2(z.x), fast_exp2(z.y));
              sum = __fadd2_rn(sum, __fadd2_rn(y, z));
            }
          }
        } else if (some) {
          const int j = slot - it.old;  // the key's place among the new tokens
#pragma unroll 1
          for (int q = 0; q < groups; ++q) {
            uint32_t sees;  // rows of the group that see the key
            if (!a.tree) {
              const int first = f - q * kGroup;
              sees = first <= 0 ? 0xFFFFFFFFu : first >= kGroup ? 0u : 0xFFFFFFFFu << first;
            } else {
              sees = j < 0 ? 0xFFFFFFFFu : 0u;
              for (int k = 0; j >= 0 && (j >> 5) < a.words && k < kGroup; ++k) {
                const int i = min((r0 + q * kGroup + k) / R, it.n - 1);  // (rows behind the last weigh nothing)
                sees |= ((*(a.tree + (it.begin + i) * a.tree_st + (j >> 5)) >> (j & 31)) & 1u) << k;
              }
            }
            float s[kGroup];
            tmem_ld32f(ts + buf * 2 * kTileRows + q * kGroup, s);
            tmem_wait_ld32(s);
            __syncwarp();
#pragma unroll
            for (int k = 0; k < kGroup; ++k) {
              const int r = side * kHalf + q * kGroup + k;
              const float y = fast_exp2(fmaf(s[k], cst[kTileRows + r] * ks, cst[r]));
              if ((sees >> k) & 1u) (k & 1 ? sum.y : sum.x) += y;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        mbar_arrive_elect(s_empty[buf]);
        mbar_arrive_elect(c_empty[cs]);
        if ((t + 1 - it.t0) % kFoldTiles == 0) {
          total += sum.x + sum.y;
          sum = make_float2(0.f, 0.f);
        }
      }
      if (alive && row != kNoRow)  // (a slot of the sequence, with memory)
        w.partial[it.partial + (side ? w.places : 0) + (a.by_pool ? row : (uint32_t)key)] = total + (sum.x + sum.y);
    }
  } else if (warp < kSumWarps + kWideWarps) {
    // ------------------------------------------------------------ keys to f16
    constexpr int CH = D / 16, KPS = 32 * kWideWarps / CH, STEPS = kKeys / KPS, FLY = 8;  // chunks of a key, keys of a step
    static_assert(STEPS == FLY || STEPS == 2 * FLY, "one or two rounds");
    const int x = tid - 32 * kSumWarps;
    const int col = CH == 8 ? (x & 3) + ((x >> 1) & 4) : x & 3;
    const int key = CH == 8 ? ((x >> 2) & 1) + 2 * (x >> 4) : x >> 2;
    const int page = a.c.page, page_log = __ffs(page) - 1;
    uint32_t items = 0;
    for (bool ok = true; ok; ++items) {
      const uint32_t kb = items % kRing;
      Item* const item = reinterpret_cast<Item*>(sm + L::oItem + kb * 64);
      if (!it.next()) {
        ok = mbar_wait(k_empty[kb], ((items / kRing) & 1) ^ 1, kErr | 9, abort);
        if (__all_sync(0xffffffffu, ok)) {
          if (x == 0) item->t0 = item->t1 = 0;
          __syncwarp();
          mbar_arrive_elect(k_full[kb]);
        }
        break;
      }
      auto page_of = [&](int i) {
        const int slot = it.k0 + i;
        return slot < it.lim ? paged_page(a.c, it.b, slot >> page_log) : -1;
      };
      float ks[2];
      uint32_t rows[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int q = page_of(x + 128 * i);
        ks[i] = q >= 0 ? a.c.k_scale[(int64_t)q * G + it.g] : 0.f;
        rows[i] = q >= 0 ? ((uint32_t)q * G + it.g) * page + ((it.k0 + x + 128 * i) & (page - 1)) : kNoRow;
      }
      int pid[FLY] = {};
      uint4 c[FLY];
      auto fetch = [&](int i, int step) {
        const int at = (it.k0 + key + KPS * step) & (page - 1);
        c[i] = make_uint4(0u, 0u, 0u, 0u);
        if (pid[i] >= 0)
          c[i] = *reinterpret_cast<const uint4*>(a.c.k + (((int64_t)pid[i] * G + it.g) * page + at) * D + col * 16);
      };
#pragma unroll
      for (int i = 0; i < FLY; ++i) pid[i] = page_of(key + KPS * i);
#pragma unroll
      for (int i = 0; i < FLY; ++i) fetch(i, i);
      if (STEPS > FLY) {
#pragma unroll
        for (int i = 0; i < FLY; ++i) pid[i] = page_of(key + KPS * (FLY + i));
      }
      ok = __all_sync(0xffffffffu, mbar_wait(k_empty[kb], ((items / kRing) & 1) ^ 1, kErr | 9, abort));
      if (!ok) break;
#pragma unroll 1
      for (int s0 = 0; s0 < STEPS; s0 += FLY) {
#pragma unroll
        for (int i = 0; i < FLY; ++i) {
          const int row = key + KPS * (s0 + i);
          const uint2 e = widen4<KV>(c[i].x), f = widen4<KV>(c[i].y), h = widen4<KV>(c[i].z), o = widen4<KV>(c[i].w);
          if (s0 + FLY < STEPS) fetch(i, s0 + FLY + i);  // the next ones, under the other widenings
          uint8_t* dst = sm + L::oK + (kb * 2 + (row >> 7)) * L::kKHalf + (col >> 2) * (128 * 128) + (row & 127) * 128;
          const int sub = (col & 3) * 2;
          *reinterpret_cast<uint4*>(dst + ((sub ^ (row & 7)) << 4)) = make_uint4(e.x, e.y, f.x, f.y);
          *reinterpret_cast<uint4*>(dst + (((sub + 1) ^ (row & 7)) << 4)) = make_uint4(h.x, h.y, o.x, o.y);
        }
      }
      if (x == 0) {
        item->t0 = it.t0; item->t1 = it.t1; item->k0 = it.k0; item->lim = it.lim;
        item->old = it.sq.old; item->n = it.sq.n; item->begin = it.sq.begin; item->nrows = it.nrows;
        item->partial = 2 * it.c * w.places +
                        (a.by_pool ? 0 : ((int64_t)it.b * G + it.g) * a.c.max_pages * page + it.k0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<float*>(sm + L::oScale + (kb * kKeys + x + 128 * i) * 4) = ks[i];
        *reinterpret_cast<uint32_t*>(sm + L::oRow + (kb * kKeys + x + 128 * i) * 4) = rows[i];
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_elect(k_full[kb]);
    }
  } else if (warp == kSumWarps + kWideWarps) {
    // ------------------------------------------------------------ query rows
    if (lane == 0) {
      uint32_t n = 0;
      bool ok = true;
      asm volatile("fence.proxy.async;" ::: "memory");  // the records are another grid's plain stores
      while (ok && it.next()) {
        const uint8_t* rec = w.tiles + (it.g * w.tiles_g + first_tile(it.sq, R, it.b)) * (int64_t)L::kRecord;
        for (int t = it.t0; t < it.t1; ++t) {
          const uint32_t qs = n % kRing, cs = n % kConsts;
          ok = mbar_wait(q_empty[qs], ((n / kRing) & 1) ^ 1, kErr | 3, abort) &&
               mbar_wait(c_empty[cs], ((n / kConsts) & 1) ^ 1, kErr | 4, abort);
          if (!ok) break;
          const uint8_t* src = rec + (int64_t)t * L::kRecord;
          mbar_arrive_expect_tx(q_full[qs], L::kQBytes);
          bulk_load(smem_u32(sm + L::oQ + qs * L::kQBytes), src, L::kQBytes, q_full[qs]);
          mbar_arrive_expect_tx(c_full[cs], kConstBytes);
          bulk_load(smem_u32(sm + L::oC + cs * kConstBytes), src + L::kQBytes, kConstBytes, c_full[cs]);
          ++n;
        }
      }
      // no copy is under way when the CTA leaves (they are long done unless a wait ran out)
      const long long start = clock64();
      for (uint32_t i = n > (uint32_t)kConsts ? n - kConsts : 0; i < n; ++i) {
        while (i + kRing >= n && !mbar_try_wait(q_full[i % kRing], (i / kRing) & 1) && clock64() - start < kWaitLimitCycles) {
        }
        while (!mbar_try_wait(c_full[i % kConsts], (i / kConsts) & 1) && clock64() - start < kWaitLimitCycles) {
        }
      }
    }
  } else {
    // ------------------------------------------------------------ MMA issue
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(1, 0, 0, 0, 128, kTileRows);
      uint32_t n = 0, items = 0;
      bool ok = true;
      while (ok) {
        const uint32_t kb = items % kRing;
        ok = mbar_wait(k_full[kb], (items / kRing) & 1, kErr | 5, abort);
        if (!ok) break;
        const int2 tiles = *reinterpret_cast<const int2*>(sm + L::oItem + kb * 64);
        if (tiles.x == tiles.y) break;
        for (int t = tiles.x; t < tiles.y && ok; ++t, ++n) {
          const uint32_t qs = n % kRing, buf = n & 1;
          ok = mbar_wait(s_empty[buf], ((n >> 1) & 1) ^ 1, kErr | 6, abort) &&
               mbar_wait(q_full[qs], (n / kRing) & 1, kErr | 7, abort);
          if (!ok) break;
          tc_fence_after();
          const uint64_t q = smem_desc_sw128(smem_u32(sm + L::oQ + qs * L::kQBytes), 16, 1024);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint64_t k = smem_desc_sw128(smem_u32(sm + L::oK + (kb * 2 + h) * L::kKHalf), 16, 1024);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {  // the descriptors' addresses count 16 bytes
              const uint32_t at = ((i >> 2) * (128 * 128) + (i & 3) * 32) >> 4;
              mma_f16(tmem + (buf * 2 + h) * kTileRows, k + at, q + at, idesc, i > 0);
            }
          }
          mma_commit(s_full[buf]);
          mma_commit(q_empty[qs]);
        }
        if (ok) mma_commit(k_empty[kb]);
        ++items;
      }
      // every MMA issued has completed before the tensor memory is freed
      mma_commit(drain);
      const long long start = clock64();
      while (!mbar_try_wait(drain, 0) && clock64() - start < kWaitLimitCycles) {
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSumWarps + kWideWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The chunks' sums into the weights.
__global__ void __launch_bounds__(kSlotThreads) paged_weigh_sum_kernel(const PagedWeighParams p, const WeighPlan w,
                                                                       int heads) {
  grid_dependents();
  grid_wait();
  const PagedAttendParams& a = p.a;
  const int b = blockIdx.y, G = a.c.G, R = a.b.H / G, g0 = blockIdx.z * heads;
  const PagedSeq sq = paged_seq(a.b, a.c, b);
  const int nrows = sq.n * R;
  WeighSlots x;
  if (nrows <= p.rows_over || !x.set(p, sq, b, blockIdx.x * kSlotsCta + kQuad * threadIdx.x)) return;
  const int c1 = (nrows + w.chunk - 1) / w.chunk;
  const SlotPlaces place(a, b, x.slot, x.row);
#pragma unroll 2
  for (int h = 0; h < min(heads, G - g0); ++h) {
    const int g = g0 + h;
    const float4 was = x.before(p, g);
    float add[kQuad] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int c = 0; c < c1; ++c) {
      const float* at = w.partial + 2 * c * w.places + place.first + g * place.head;
      const float4 y = *reinterpret_cast<const float4*>(at), z = *reinterpret_cast<const float4*>(at + w.places);
      const float part[kQuad] = {y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w};
      // a chunk of which no row sees a slot has left nothing for it
      const int64_t seen = a.tree ? INT64_MAX : (int64_t)x.old + ((int64_t)min((c + 1) * w.chunk, nrows) - 1) / R + 1;
#pragma unroll
      for (int i = 0; i < kQuad; ++i) add[i] += x.slot + i < seen ? part[i] : 0.f;
    }
    x.finish(p, sq, g, was, add);
  }
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

int64_t most_rows(const PagedWeighParams& p) { return (int64_t)p.a.b.max_tokens * (p.a.b.H / p.a.c.G); }

// Chunks of 768 rows, up to 32 of them, in at most 1 GiB of sums (8 bytes a chunk and place; one
// chunk there is always, whatever the places): an item's keys cost
// about as much to widen as two tiles of rows to multiply and sum (1024 new tokens over 8192, 2
// sequences: 313, 279, 263, 259 and 262 us with 256, 384, 512, 768 and 1024 rows).
size_t plan_for(const PagedWeighParams& p, void* ws, WeighPlan& x) {
  const PagedAttendParams& a = p.a;
  const int64_t rows = most_rows(p);
  x.places = slot_places(a, a.by_pool);
  const int64_t fit = std::max<int64_t>(1, ((int64_t)1 << 27) / x.places);
  const int64_t most = std::min<int64_t>(std::min<int64_t>(32, fit), (rows + 767) / 768);
  x.chunk = (int)((rows + most * kTileRows - 1) / (most * kTileRows) * kTileRows);
  x.chunks = (int)((rows + x.chunk - 1) / x.chunk);
  x.tiles_g = (int64_t)a.b.T * (a.b.H / a.c.G) / kTileRows + a.b.B + 1;
  uint8_t* w = static_cast<uint8_t*>(ws);
  const size_t tiles = align256((size_t)x.tiles_g * a.c.G * (a.c.D == 128 ? Lay<128>::kRecord : Lay<64>::kRecord));
  x.tiles = w;
  x.partial = reinterpret_cast<float*>(w + (w ? tiles : 0));
  return tiles + align256((size_t)x.chunks * 2 * x.places * sizeof(float));
}

template <int KV, int D>
cudaError_t tc_launch(const PagedWeighParams& p, bool bf16, const WeighPlan& w, int n_sm, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may use its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
    e = cudaFuncSetAttribute(paged_weigh_tc_kernel<KV, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Lay<D>::bytes(paged_attend_max_batch()));
    if (e != cudaSuccess) return e;
    if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const PagedAttendParams& a = p.a;
  const dim3 tiles((unsigned)w.tiles_g, a.c.G);
  e = launch_dependent(paged_weigh_rows_kernel<D>, tiles, kRowThreads, 0, st, p, w, bf16);
  if (e != cudaSuccess) return e;
  const int64_t slots = (int64_t)a.c.max_pages * a.c.page;
  const double items = (double)a.b.B * a.c.G * w.chunks * ((slots + kKeys - 1) / kKeys);
  e = launch_dependent(paged_weigh_tc_kernel<KV, D>, dim3((unsigned)std::min((double)n_sm, items)), kThreads,
                       Lay<D>::bytes(a.b.B), st, p, w);
  if (e != cudaSuccess) return e;
  int heads;
  const dim3 grid = slot_grid(p, n_sm, kSlotsCta, heads);
  return launch_dependent(paged_weigh_sum_kernel, grid, kSlotThreads, 0, st, p, w, heads);
}

bool many_rows(const PagedWeighParams& p) { return most_rows(p) > p.rows_over; }

}  // namespace

size_t paged_weigh_workspace(const PagedWeighParams& p) {
  WeighPlan x;
  return many_rows(p) ? plan_for(p, nullptr, x) : 0;
}

cudaError_t launch_paged_weigh(const PagedWeighParams& p, int dtype, int kv, void* ws, int n_sm, cudaStream_t st) {
  if (dtype != kF16 && dtype != kBF16) return cudaErrorInvalidValue;
  if (p.a.score) {
    const cudaError_t e = scores_launch(p, n_sm, st);
    if (e != cudaSuccess) return e;
  }
  if (!many_rows(p)) return cudaSuccess;
  WeighPlan x;
  plan_for(p, ws, x);
  const bool bf16 = dtype == kBF16;
  if (p.a.c.D == 128)
    return kv == kKvInt8 ? tc_launch<kKvInt8, 128>(p, bf16, x, n_sm, st) : tc_launch<kKvE4m3, 128>(p, bf16, x, n_sm, st);
  if (p.a.c.D == 64)
    return kv == kKvInt8 ? tc_launch<kKvInt8, 64>(p, bf16, x, n_sm, st) : tc_launch<kKvE4m3, 64>(p, bf16, x, n_sm, st);
  return cudaErrorInvalidValue;
}

cudaError_t read_paged_weigh_error(unsigned int* code, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(code, sm100::g_device_error, sizeof(unsigned int));
  if (e != cudaSuccess || !reset) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(sm100::g_device_error, &zero, sizeof(unsigned int));
}

}  // namespace spatten
