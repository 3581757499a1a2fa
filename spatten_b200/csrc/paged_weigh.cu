// The weights that the new tokens give the cached ones (spatten_paged_attend_ext
// with weights): after the attention, whose statistics (m, 1 / l) of each row are
// read,
//   weight[slot] = (slot is an earlier token's ? weight[slot] : 0) + sum over rows
//                  of 2^(q . k sm_scale log2(e) - m) / l
// for every slot that a row of the call may see; the new tokens' slots take their
// positions. Two ways, by the query rows that a sequence has per KV head:
//
// Up to kScoreRows: the attention has kept its scores (4 bytes a row and slot), and
// paged_weigh_scores_kernel, a thread per slot, turns them into weights. For 64
// sequences x 8 heads x 32768 keys with 4 rows this reads and writes 470 MB; reading
// the keys again would take 2.1 GB.
//
// More: the scores are computed again, on the tensor cores, with the keys as rows:
//   S^T [128 keys x 64 rows] = K codes . Q'^T   (kind::f16, fp32 in tensor memory),
// so that a thread owns a key and the sum over rows needs no exchange.
// paged_weigh_rows_kernel lays the query rows out once (f16 as the attention's, in
// the layout that the MMAs read, and two numbers a row: cq, its scores' factor, and
// b = log2(1 / l) - m, so that p = 2^(S (cq k_scale) + b)); paged_weigh_tc_kernel
// takes 256 keys x a chunk of the rows at a time; the last kernel adds the chunks up.
// Bound by the exponentials, one per (row, key).
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

// Slots x sequences x groups of heads; groups of `heads`, smaller where the CTAs are few.
dim3 slot_grid(const PagedWeighParams& p, int n_sm, int& heads) {
  const int64_t slots = (int64_t)p.a.c.max_pages * p.a.c.page, G = p.a.c.G;
  const int64_t ctas = (slots + kSlotsCta - 1) / kSlotsCta;
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
  if (tid < heads * ROWS && g0 + tid / ROWS < G) {
    const int g = g0 + tid / ROWS, r = tid % ROWS;
    if (r < nrows) stat[tid / ROWS][r] = a.stat[(int64_t)(sq.begin + r / R) * a.b.H + g * R + r % R];
  }
  __syncthreads();
  if (!live) return;
  const int64_t slots = (int64_t)a.c.max_pages * a.c.page;
  const float* src = a.score + ((int64_t)b * G * slots + x.slot) * ROWS;
#pragma unroll 2
  for (int h = 0; h < min(heads, G - g0); ++h) {
    const int g = g0 + h;
    float s[kQuad * ROWS];
    const float4* at = reinterpret_cast<const float4*>(src + g * slots * ROWS);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const float4 y = at[i];
      s[4 * i] = y.x; s[4 * i + 1] = y.y; s[4 * i + 2] = y.z; s[4 * i + 3] = y.w;
    }
    const float4 was = x.before(p, g);
    float add[kQuad] = {0.f, 0.f, 0.f, 0.f};
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

cudaError_t scores_launch(const PagedWeighParams& p, int n_sm, cudaStream_t st) {
  int heads;
  const dim3 grid = slot_grid(p, n_sm, heads);
  switch (p.a.score_rows) {
    case 1: return launch_dependent(paged_weigh_scores_kernel<1>, grid, kSlotThreads, 0, st, p, heads);
    case 2: return launch_dependent(paged_weigh_scores_kernel<2>, grid, kSlotThreads, 0, st, p, heads);
    case 4: return launch_dependent(paged_weigh_scores_kernel<4>, grid, kSlotThreads, 0, st, p, heads);
    case 8: return launch_dependent(paged_weigh_scores_kernel<8>, grid, kSlotThreads, 0, st, p, heads);
    default: return cudaErrorInvalidValue;
  }
}

// ---------------------------------------------------------------- many rows: tensor cores

constexpr int kKeys = 256, kTileRows = 64, kFoldTiles = 8;
constexpr int kSumWarps = 8, kThreads = 32 * (kSumWarps + 2);
constexpr int kConsts = 4;               // tiles' row constants in shared memory
constexpr int kConstBytes = kTileRows * 8;
constexpr unsigned kErr = 0x500;

// What the main kernel works on, in the workspace.
struct WeighPlan {
  uint8_t* tiles;     // [G][tiles_g] records: 64 query rows, then their constants
  float* partial;     // [chunks][B][G][slots]
  int64_t tiles_g;
  int chunk, chunks;  // rows of a chunk (a multiple of kTileRows), chunks of a sequence at most
};

template <int D>
struct Lay {
  static constexpr int kRing = D == 128 ? 2 : 4;            // tiles of query rows
  static constexpr int kQBytes = kTileRows * D * 2;
  static constexpr int kRecord = kQBytes + kConstBytes;
  static constexpr int oK = 0;                               // [2][D / 64][128][128 B]
  static constexpr int kKHalf = 128 * D * 2;
  static constexpr int oQ = oK + 2 * kKHalf;                 // [ring][D / 64][64][128 B]
  static constexpr int oC = oQ + kRing * kQBytes;            // [kConsts][32][cq, cq, b, b]
  static constexpr int oBar = oC + kConsts * kConstBytes;
  static constexpr int kBars = 2 * kRing + 2 * kConsts + 2 + 2 + 1 + 1;
  static constexpr int oTmem = oBar + kBars * 8;
  static constexpr int oAbort = oTmem + 4;
  static constexpr int oScan = (oAbort + 4 + 7) & ~7;        // [10] 64-bit
  static constexpr int oPre = oScan + 8 * (kThreads / 32);   // [B + 1]
  static constexpr int bytes(int B) { return oPre + (B + 1) * 4 + 1024; }
};

// First record of sequence b: records of sequences whose rows are apart are apart.
SPATTEN_DEV int64_t first_tile(const PagedSeq& s, int R, int b) { return (int64_t)s.begin * R / kTileRows + b; }

template <int D>
__global__ void __launch_bounds__(256) paged_weigh_rows_kernel(const PagedWeighParams p, const WeighPlan w, bool bf16) {
  using L = Lay<D>;
  constexpr int LQ = D / 8, RPP = 256 / LQ;  // lanes of a row, rows of a pass
  grid_dependents();
  grid_wait();
  const PagedAttendParams& a = p.a;
  const int b = blockIdx.z, g = blockIdx.y, t = blockIdx.x, R = a.b.H / a.c.G, tid = threadIdx.x;
  const PagedSeq sq = paged_seq(a.b, a.c, b);
  const int nrows = sq.n * R;
  if (nrows <= p.rows_over || t * kTileRows >= nrows) return;
  uint8_t* rec = w.tiles + (g * w.tiles_g + first_tile(sq, R, b) + t) * (int64_t)L::kRecord;
  const int li = tid % LQ;
  auto pair = [&](uint32_t x) {
    return bf16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u))
                : __half22float2(*reinterpret_cast<const __half2*>(&x));
  };
  uint4 x[kTileRows / RPP];
#pragma unroll
  for (int k = 0; k < kTileRows / RPP; ++k) {
    const int r = t * kTileRows + k * RPP + tid / LQ;
    x[k] = make_uint4(0u, 0u, 0u, 0u);
    if (r < nrows)
      x[k] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (int64_t)(sq.begin + r / R) * a.q_st +
                                             (int64_t)(g * R + r % R) * a.q_sh + 8 * li);
  }
#pragma unroll
  for (int k = 0; k < kTileRows / RPP; ++k) {
    const int y = k * RPP + tid / LQ, r = t * kTileRows + y;
    const uint32_t in[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = pair(in[j]);
      top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      if (!(f.x == f.x && f.y == f.y)) top = INFINITY;  // fmaxf drops a NaN
    }
#pragma unroll
    for (int d = LQ / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const QueryScale qs = query_scale(top, a.scale_log2);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = pair(in[j]);
      o[j] = pack2<__half>(f.x * qs.up, f.y * qs.up);
    }
    *reinterpret_cast<uint4*>(rec + (li >> 3) * (kTileRows * 128) + y * 128 + (((li & 7) ^ (y & 7)) << 4)) =
        make_uint4(o[0], o[1], o[2], o[3]);
    if (li == 0) {
      float2 c = make_float2(0.f, -INFINITY);  // no row: no weight
      if (r < nrows) {
        const float2 s = a.stat[(int64_t)(sq.begin + r / R) * a.b.H + g * R + r % R];
        c = make_float2(qs.factor, log2f(s.y) - s.x);
      }
      float* to = reinterpret_cast<float*>(rec + L::kQBytes) + (y >> 1) * 4 + (y & 1);
      to[0] = c.x;
      to[2] = c.y;
    }
  }
}

SPATTEN_DEV void bulk_load(uint32_t dst, const void* src, uint32_t bytes, SBar bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar.a)
               : "memory");
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

// The items of a CTA: 256 keys of a (sequence, KV head) by a chunk of its rows.
// Every role walks them by itself.
struct Items {
  const PagedWeighParams& p;
  const WeighPlan& w;
  const uint32_t* pre;
  uint32_t next_item, total;
  // the item
  PagedSeq sq;
  int b, g, c, k0, lim, nrows, t0, t1;  // row tiles [t0, t1)

  static SPATTEN_DEV int limit(const PagedSeq& s) { return max(min(s.old + s.n, s.len), 0); }
  static SPATTEN_DEV unsigned long long count(const PagedWeighParams& p, const WeighPlan& w, int b) {
    const PagedSeq s = paged_seq(p.a.b, p.a.c, b);
    const int R = p.a.b.H / p.a.c.G, rows = s.n * R;
    if (rows <= p.rows_over) return 0;
    return (unsigned long long)p.a.c.G * ((rows + w.chunk - 1) / w.chunk) * ((limit(s) + kKeys - 1) / kKeys);
  }
  SPATTEN_DEV bool next() {
    while (next_item < total) {
      const uint32_t u = next_item;
      next_item += gridDim.x;
      int lo = 0;
      for (int hi = p.a.b.B; hi - lo > 1;) {  // the sequence of item u
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= u) lo = mid; else hi = mid;
      }
      b = lo;
      sq = paged_seq(p.a.b, p.a.c, b);
      const int R = p.a.b.H / p.a.c.G;
      lim = limit(sq);
      nrows = sq.n * R;
      const uint32_t kt = (lim + kKeys - 1) / kKeys, ch = (nrows + w.chunk - 1) / w.chunk, x = u - pre[b];
      k0 = (int)(x % kt) * kKeys;
      c = (int)(x / kt % ch);
      g = (int)(x / kt / ch);
      t0 = c * (w.chunk / kTileRows);
      t1 = min(t0 + w.chunk / kTileRows, (nrows + kTileRows - 1) / kTileRows);
      if (!p.a.tree && k0 > sq.old) t0 = max(t0, (int)min((int64_t)(k0 - sq.old) * R / kTileRows, (int64_t)INT_MAX));
      if (t0 < t1) return true;
    }
    return false;
  }
};

template <int KV, int D>
__global__ void __launch_bounds__(kThreads, 2) paged_weigh_tc_kernel(const PagedWeighParams p, const WeighPlan w) {
  using L = Lay<D>;
  constexpr int RING = L::kRing;
  extern __shared__ uint8_t smem_raw[];
  grid_dependents();
  grid_wait();
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t bars = smem_u32(sm + L::oBar);
  const SBarArr q_full{bars}, q_empty{bars + 8 * RING}, c_full{bars + 16 * RING},
      c_empty{bars + 16 * RING + 8 * kConsts}, s_full{bars + 16 * RING + 16 * kConsts},
      s_empty{bars + 16 * RING + 16 * kConsts + 16}, rest{bars + 16 * RING + 16 * kConsts + 32};
  const SBar k_full = rest[0], drain = rest[1];
  volatile int* abort = reinterpret_cast<volatile int*>(sm + L::oAbort);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + L::oTmem);
  uint32_t* pre = reinterpret_cast<uint32_t*>(sm + L::oPre);
  unsigned long long* scan = reinterpret_cast<unsigned long long*>(sm + L::oScan);
  const PagedAttendParams& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.c.G, R = a.b.H / G;

  if (tid == 0) {
    for (int i = 0; i < RING; ++i) {
      mbar_init(q_full[i], 1);
      mbar_init(q_empty[i], 1);
    }
    for (int i = 0; i < kConsts; ++i) {
      mbar_init(c_full[i], 1);
      mbar_init(c_empty[i], kSumWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full[i], 1);
      mbar_init(s_empty[i], kSumWarps);
    }
    mbar_init(k_full, kSumWarps);
    mbar_init(drain, 1);
    fence_barrier_init();
    *abort = 0;
    pre[0] = 0;
  }
  if (warp == kSumWarps + 1) {
    tmem_alloc(tslot, 256);
    tmem_relinquish();
  }
  unsigned long long U = 0;
  for (int base = 0; base < a.b.B; base += kThreads) {
    const int b = base + tid;
    unsigned long long x = b < a.b.B ? Items::count(p, w, b) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    unsigned long long front = U;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) front += scan[i];
      U += scan[i];
    }
    if (b < a.b.B) pre[b + 1] = (uint32_t)(front + x);
    __syncthreads();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  // (the attention's host check leaves 32 bits for sequences that share no rows)
  Items it{p, w, pre, blockIdx.x, U >> 32 ? 0u : (uint32_t)U};

  if (warp < kSumWarps) {
    // ------------------------------------------------------------ keys to f16, sums of the weights
    constexpr int CH = D / 16, KPS = 32 * kSumWarps / CH, STEPS = kKeys / KPS;  // chunks of a key, keys of a step
    const int col = CH == 8 ? (tid & 3) + ((tid >> 1) & 4) : tid & 3;
    const int key = CH == 8 ? ((tid >> 2) & 1) + 2 * (tid >> 4) : tid >> 2;
    const int page = a.c.page, page_log = __ffs(page) - 1;
    const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (warp >> 2) * kTileRows;
    uint32_t n = 0;  // tiles
    bool alive = true;
    while (alive && it.next()) {
      // (the item before is through: its last scores were there)
      int pid[STEPS];
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int slot = it.k0 + key + KPS * i;
        pid[i] = slot < it.lim ? paged_page(a.c, it.b, slot >> page_log) : -1;
      }
      const int slot = it.k0 + tid;
      const int pid_s = slot < it.lim ? paged_page(a.c, it.b, slot >> page_log) : -1;
      uint4 x[STEPS];
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int at = (it.k0 + key + KPS * i) & (page - 1);
        x[i] = make_uint4(0u, 0u, 0u, 0u);
        if (pid[i] >= 0)
          x[i] = *reinterpret_cast<const uint4*>(a.c.k + (((int64_t)pid[i] * G + it.g) * page + at) * D + col * 16);
      }
      const float ks = pid_s >= 0 ? a.c.k_scale[(int64_t)pid_s * G + it.g] : 0.f;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int row = key + KPS * i;
        const uint2 e = widen4<KV>(x[i].x), f = widen4<KV>(x[i].y), h = widen4<KV>(x[i].z), o = widen4<KV>(x[i].w);
        uint8_t* dst = sm + L::oK + (row >> 7) * L::kKHalf + (col >> 2) * (128 * 128) + (row & 127) * 128;
        const int sub = (col & 3) * 2;
        *reinterpret_cast<uint4*>(dst + ((sub ^ (row & 7)) << 4)) = make_uint4(e.x, e.y, f.x, f.y);
        *reinterpret_cast<uint4*>(dst + (((sub + 1) ^ (row & 7)) << 4)) = make_uint4(h.x, h.y, o.x, o.y);
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_elect(k_full);

      const float2 ks2 = make_float2(ks, ks);
      float total = 0.f;
      float2 sum = make_float2(0.f, 0.f);
      const int last = min(it.k0 + (warp << 5) + 31, it.lim - 1);  // key of the warp
      for (int t = it.t0; t < it.t1; ++t, ++n) {
        const uint32_t buf = n & 1, cs = n % kConsts;
        bool ok = mbar_wait(s_full[buf], (n >> 1) & 1, kErr | 1, abort);
        ok = ok && mbar_wait(c_full[cs], (n / kConsts) & 1, kErr | 2, abort);
        if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        tc_fence_after();
        float s[kTileRows];
        tmem_ld32f(ts + buf * 128, s);
        tmem_ld32f(ts + buf * 128 + 32, s + 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_elect(s_empty[buf]);
        const float4* cst = reinterpret_cast<const float4*>(sm + L::oC + cs * kConstBytes);
        const int r0 = t * kTileRows;
        const int sees = it.sq.old + (a.tree ? 0 : r0 / R + 1);  // slots before it are seen by every row of the tile
        auto weights2 = [&](int k) {  // of rows 2 k and 2 k + 1
          const float4 c = cst[k];
          const float2 y = __ffma2_rn(make_float2(s[2 * k], s[2 * k + 1]), __fmul2_rn(make_float2(c.x, c.y), ks2),
                                      make_float2(c.z, c.w));
          return make_float2(fast_exp2(y.x), fast_exp2(y.y));
        };
        if (last < sees) {
#pragma unroll
          for (int k = 0; k < kTileRows / 2; ++k) sum = __fadd2_rn(sum, weights2(k));
        } else if (!a.tree) {
          // the first row of the tile that sees the key
          const int64_t first = max((int64_t)(slot - it.sq.old) * R - r0, (int64_t)0);
          if (__any_sync(0xffffffffu, first < kTileRows)) {
            const int f = (int)min(first, (int64_t)kTileRows);
#pragma unroll
            for (int k = 0; k < kTileRows / 2; ++k) {
              const float2 y = weights2(k);
              sum = __fadd2_rn(sum, make_float2(2 * k >= f ? y.x : 0.f, 2 * k + 1 >= f ? y.y : 0.f));
            }
          }
        } else {
          const int j = slot - it.sq.old;  // the key's place among the new tokens
          const bool none = (j >> 5) >= a.words;
#pragma unroll
          for (int k = 0; k < kTileRows / 2; ++k) {
            const float2 y = weights2(k);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int i = min((r0 + 2 * k + h) / R, it.sq.n - 1);  // (rows behind the last one weigh nothing)
              bool see = j < 0;
              if (!see && !none) see = (*(a.tree + (it.sq.begin + i) * a.tree_st + (j >> 5)) >> (j & 31)) & 1u;
              if (see) (h ? sum.y : sum.x) += h ? y.y : y.x;
            }
          }
        }
        __syncwarp();
        mbar_arrive_elect(c_empty[cs]);
        if ((t + 1 - it.t0) % kFoldTiles == 0) {
          total += sum.x + sum.y;
          sum = make_float2(0.f, 0.f);
        }
      }
      if (alive && slot < it.lim)
        w.partial[(((int64_t)it.c * a.b.B + it.b) * G + it.g) * a.c.max_pages * page + slot] = total + (sum.x + sum.y);
    }
  } else if (warp == kSumWarps) {
    // ------------------------------------------------------------ query rows
    if (lane == 0) {
      uint32_t n = 0;
      bool ok = true;
      asm volatile("fence.proxy.async;" ::: "memory");  // the records are another grid's plain stores
      while (ok && it.next()) {
        const uint8_t* rec = w.tiles + (it.g * w.tiles_g + first_tile(it.sq, R, it.b)) * (int64_t)L::kRecord;
        for (int t = it.t0; t < it.t1; ++t) {
          const uint32_t qs = n % RING, cs = n % kConsts;
          ok = mbar_wait(q_empty[qs], ((n / RING) & 1) ^ 1, kErr | 3, abort) &&
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
        while (i + RING >= n && !mbar_try_wait(q_full[i % RING], (i / RING) & 1) && clock64() - start < kWaitLimitCycles) {
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
      while (ok && it.next()) {
        ok = mbar_wait(k_full, items++ & 1, kErr | 5, abort);
        for (int t = it.t0; t < it.t1 && ok; ++t, ++n) {
          const uint32_t qs = n % RING, buf = n & 1;
          ok = mbar_wait(s_empty[buf], ((n >> 1) & 1) ^ 1, kErr | 6, abort) &&
               mbar_wait(q_full[qs], (n / RING) & 1, kErr | 7, abort);
          if (!ok) break;
          tc_fence_after();
          const uint64_t q = smem_desc_sw128(smem_u32(sm + L::oQ + qs * L::kQBytes), 16, 1024);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint64_t k = smem_desc_sw128(smem_u32(sm + L::oK + h * L::kKHalf), 16, 1024);
#pragma unroll
            for (int i = 0; i < D / 16; ++i)  // the descriptors' addresses count 16 bytes
              mma_f16(tmem + buf * 128 + h * kTileRows, k + (((i >> 2) * (128 * 128) + (i & 3) * 32) >> 4),
                      q + (((i >> 2) * (kTileRows * 128) + (i & 3) * 32) >> 4), idesc, i > 0);
          }
          mma_commit(s_full[buf]);
          mma_commit(q_empty[qs]);
        }
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
  if (warp == kSumWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
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
  const int64_t slots = (int64_t)a.c.max_pages * a.c.page;
#pragma unroll 2
  for (int h = 0; h < min(heads, G - g0); ++h) {
    const int g = g0 + h;
    const float4 was = x.before(p, g);
    float add[kQuad] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int c = 0; c < c1; ++c) {
      const float4 y = *reinterpret_cast<const float4*>(w.partial + (((int64_t)c * a.b.B + b) * G + g) * slots + x.slot);
      const float part[kQuad] = {y.x, y.y, y.z, y.w};
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

// Chunks of at least 512 rows, up to eight of them, in at most 1 GiB of sums.
size_t plan_for(const PagedWeighParams& p, void* ws, WeighPlan& x) {
  const PagedAttendParams& a = p.a;
  const int64_t rows = most_rows(p), slots = (int64_t)a.c.max_pages * a.c.page;
  const int64_t fit = std::max<int64_t>(1, ((int64_t)1 << 28) / std::max<int64_t>(1, slots * a.b.B * a.c.G));
  const int64_t most = std::min<int64_t>(std::min<int64_t>(8, fit), (rows + 511) / 512);
  x.chunk = (int)((rows + most * kTileRows - 1) / (most * kTileRows) * kTileRows);
  x.chunks = (int)((rows + x.chunk - 1) / x.chunk);
  x.tiles_g = (int64_t)a.b.T * (a.b.H / a.c.G) / kTileRows + a.b.B + 1;
  uint8_t* w = static_cast<uint8_t*>(ws);
  const size_t tiles = align256((size_t)x.tiles_g * a.c.G * (a.c.D == 128 ? Lay<128>::kRecord : Lay<64>::kRecord));
  x.tiles = w;
  x.partial = reinterpret_cast<float*>(w + (w ? tiles : 0));
  return tiles + align256((size_t)x.chunks * a.b.B * a.c.G * slots * sizeof(float));
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
  const dim3 tiles((unsigned)((most_rows(p) + kTileRows - 1) / kTileRows), a.c.G, a.b.B);
  e = launch_dependent(paged_weigh_rows_kernel<D>, tiles, 256, 0, st, p, w, bf16);
  if (e != cudaSuccess) return e;
  const int64_t slots = (int64_t)a.c.max_pages * a.c.page;
  const double items = (double)a.b.B * a.c.G * w.chunks * ((slots + kKeys - 1) / kKeys);
  e = launch_dependent(paged_weigh_tc_kernel<KV, D>, dim3((unsigned)std::min(2.0 * n_sm, items)), kThreads,
                       Lay<D>::bytes(a.b.B), st, p, w);
  if (e != cudaSuccess) return e;
  int heads;
  const dim3 grid = slot_grid(p, n_sm, heads);
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
