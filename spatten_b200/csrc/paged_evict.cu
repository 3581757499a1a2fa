// Tokens that leave the paged 8-bit KV cache: eviction by accumulated attention
// weight (spatten_paged_evict), and the rejected ones among drafted tokens
// (spatten_paged_keep).
//
// Eviction. A sequence of more than `keep` slots keeps the tokens of the `recent`
// newest positions, then those of the largest weight, ties to the lower slot. Its
// kept tokens in slots behind `keep` move into the free slots before it, both in
// ascending order. Nothing else moves: what is read (slots from `keep` on) and what is
// written (slots before) are apart, so every written block is a CTA of its own, and
// a token is rounded again only when it moves. Three launches:
//
// paged_rank_kernel: the slots' keys, out of the pages.
//
// paged_select_kernel: a cluster of CTAs per sequence (or per sequence and KV head),
// each holding the ordered keys of a run of slots in shared memory. The keep-th
// largest key by radix rounds of 11 bits, whose histograms are summed over the
// cluster; then the kept, the free and the moving slots as bits, a word per 32 slots,
// whose prefix sums number them.
//
// paged_move_kernel: a CTA per block (page, KV head) of the first `keep` slots. A
// token's codes under the block's scale S' are round(code * S / S') with S' the larger of the block's scale (0 where it keeps nothing) and the one that the
// largest moved magnitude needs; where S' grew, the kept codes are rounded likewise, as
// appending does.
//
// Bound by latency, the chain of loads and of cluster barriers: 131001 slots of one
// sequence cut to 65536 62 us (the moved codes alone are 134 MB, 21 us), 48 sequences of up
// to 5000 slots cut to 4096 by head 72 us, 16 of 1088 cut to 1024 25 us. With the keys
// gathered by the selection itself (8 CTAs for the longest case) that took 123 us of its
// own; the selection's code, which runs once, is kept small (28 -> 25 us).
#include <atomic>
#include <cooperative_groups.h>

#include "kernels.h"
#include "paged_dev.cuh"

namespace cg = cooperative_groups;

namespace spatten {
namespace {

constexpr float kMaxFinite = 3.402823466e38f;
constexpr uint32_t kNoRow = 0xFFFFFFFFu;

// ---------------------------------------------------------------- moving rows

template <int D, int PAGE>
struct MoveShape {
  static constexpr int LPR = D / 16;                                 // lanes per row
  static constexpr int NT = PAGE * LPR < 256 ? 64 : PAGE * LPR / 4;  // threads, at least one a row
  static constexpr int RPP = NT / LPR;                               // rows per pass
  static constexpr int PASSES = PAGE / RPP;                          // at most 4
  static_assert(NT >= PAGE && PASSES <= 4 && PAGE % RPP == 0, "a row's move per thread, a block in registers");
};

// The rows of one block that tokens move into.
template <int PAGE>
struct MoveRows {
  uint32_t src[PAGE];     // row of the pools, kNoRow: none
  float scale[2][PAGE];   // its scales, K's and V's
  uint32_t red[2][8];
};

template <int KV>
SPATTEN_DEV float row_amax(uint4 c) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[4];
    codes4_to_f32_alu<KV>(w[i], f);
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(f[e]));
  }
  return m;
}

template <int KV>
SPATTEN_DEV uint4 rescale16(uint4 c, float ratio) {
  const uint2 a = rescale8<KV>(make_uint2(c.x, c.y), ratio), b = rescale8<KV>(make_uint2(c.z, c.w), ratio);
  return make_uint4(a.x, a.y, b.x, b.y);
}

// Moves m's rows into block `to` of K and of V, whose scales were `was` (the rows before
// `end` that get none keep their tokens, if `kept` says that there are any). All
// threads of the CTA; every source is read before anything is written.
template <int KV, int D, int PAGE>
SPATTEN_DEV void move_block(MoveRows<PAGE>& m, const PagedCache& pc, int64_t to, float2 was, bool kept, int end) {
  using S = MoveShape<D, PAGE>;
  const int tid = threadIdx.x, lane = tid & 31, li = tid % S::LPR, rt = tid / S::LPR;
  uint8_t* const pool[2] = {pc.k, pc.v};
  uint4 c[2][S::PASSES];
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int j = 0; j < S::PASSES; ++j) {
      const uint32_t row = m.src[j * S::RPP + rt];
      c[v][j] = make_uint4(0u, 0u, 0u, 0u);
      if (row != kNoRow) c[v][j] = *reinterpret_cast<const uint4*>(pool[v] + (uint64_t)row * D + li * 16);
    }
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < S::PASSES; ++j) {
      const int r = j * S::RPP + rt;
      if (m.src[r] != kNoRow) amax = fmaxf(amax, fminf(row_amax<KV>(c[v][j]) * m.scale[v][r], kMaxFinite));
    }
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));  // magnitudes order as integers
    if (lane == 0) m.red[v][tid >> 5] = top;
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    uint32_t all = 0u;
#pragma unroll
    for (int w = 0; w < S::NT / 32; ++w) all = max(all, m.red[v][w]);
    const float s_old = kept ? (v ? was.y : was.x) : 0.f, s = fmaxf(s_old, scale_for<KV>(__uint_as_float(all)));
#pragma unroll
    for (int j = 0; j < S::PASSES; ++j) {
      const int r = j * S::RPP + rt;
      uint4* at = reinterpret_cast<uint4*>(pool[v] + (to * PAGE + r) * D + li * 16);
      if (m.src[r] != kNoRow) {
        const float from = m.scale[v][r];
        // (a row of zeros asks for no scale of its own, so its ratio may overflow: 0 inf would be a NaN)
        *at = s == from ? c[v][j]
              : s > 0.f ? rescale16<KV>(c[v][j], fminf(__fdiv_rn(from, s), kMaxFinite))
                        : make_uint4(0u, 0u, 0u, 0u);
      } else if (r < end && s > s_old && kept) {
        *at = rescale16<KV>(*at, __fdiv_rn(s_old, s));
      }
    }
    if (tid == 0) (v ? pc.v_scale : pc.k_scale)[to] = s;
  }
}

// ---------------------------------------------------------------- eviction

// What the selection leaves for the moves, per sequence (and KV head): `moves`
// tokens, the i-th from slot src[base + i] to slot dst[base + i]; first[j]: moves into blocks before j.
//
// The page tables may have many times the slots of the pool (256 sequences x 8 heads, tables of
// 131072 slots beside a pool of 1.3 million: 2.2 GB for what lies by slot). Then by_pool: keys and
// positions lie like the pool (sequences that share a page have the same there), and the lists'
// places are taken as they are needed, at most one for each slot of the pool, as no two tokens move
// to the same (a call that breaks that rule leaves the sequences alone that find no place).
struct EvictPlan {
  uint32_t* head;   // [lines][4]: moves, new length, base
  int32_t* first;   // [lines][blocks + 1]
  int32_t* dst;     // [room]
  int32_t* src;     // [room]
  unsigned long long* used;  // by_pool: places taken
  float* edge;      // [B][G][2]: scales of the block of slot `keep` before the moves
  uint32_t* key;    // [lines][pitch] or [P][lines_per_b][page]: weights in the order of integers, kNoKey: no memory
  int32_t* place;   // the same of positions, where recent > 0
  int64_t room;
  int lines_per_b, blocks, cap, pitch, usable;  // usable: slots that a sequence may hold
  bool by_pool;
};

// Where a slot's key lies when they lie like the pool; negative: no memory.
SPATTEN_DEV int64_t pooled_key(const PagedCache& c, const EvictPlan& plan, int b, int hl, int slot, int page_log) {
  const int pid = paged_page(c, b, slot >> page_log);
  return pid < 0 ? -1 : (((int64_t)pid * plan.lines_per_b + hl) << page_log) + (slot & (c.page - 1));
}

// Keys of the slots, four of a page a thread. Weights that are not negative order as
// integers; negative ones and NaN count as 0.
constexpr uint32_t kNoKey = 0xFFFFFFFFu;
constexpr int kRankThreads = 128, kRankSlots = 4 * kRankThreads;

__global__ void __launch_bounds__(kRankThreads) paged_rank_kernel(const PagedEvictParams p, const EvictPlan plan) {
  grid_dependents();
  grid_wait();
  const int b = blockIdx.z, hl = blockIdx.y, slot = blockIdx.x * kRankSlots + 4 * threadIdx.x;
  const int len = *(p.lens + b), G = p.c.G, page = p.c.page;
  if (plan.by_pool && blockIdx.x == 0 && b == 0 && hl == 0 && threadIdx.x == 0) *plan.used = 0;
  if (len <= p.keep || slot >= len || len > plan.usable) return;
  const int pid = paged_page(p.c, b, slot / page);
  const int64_t row = ((int64_t)max(pid, 0) * G + hl) * page + slot % page;
  float w[4];
  if (p.per_head) {
    const float4 x = *reinterpret_cast<const float4*>(p.weight + row);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else {
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 8
    for (int g = 0; g < G; ++g) {
      const float4 x = *reinterpret_cast<const float4*>(p.weight + row + (int64_t)g * page);
      sum[0] += (double)x.x; sum[1] += (double)x.y; sum[2] += (double)x.z; sum[3] += (double)x.w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (float)sum[i];
  }
  uint32_t k[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = pid < 0 ? kNoKey : w[i] > 0.f ? __float_as_uint(w[i]) : 0u;
  const int64_t at = plan.by_pool ? ((int64_t)pid * plan.lines_per_b + hl) * page + slot % page
                                  : ((int64_t)b * plan.lines_per_b + hl) * plan.pitch + slot;
  if (at < 0) return;  // (no memory, and no place for its key)
  *reinterpret_cast<uint4*>(plan.key + at) = make_uint4(k[0], k[1], k[2], k[3]);
  if (p.recent > 0) *reinterpret_cast<int4*>(plan.place + at) = *reinterpret_cast<const int4*>(p.position + row);
}

constexpr int kSelThreads = 1024, kBins = 2048;
constexpr int kMaxWords = 40960;  // of a CTA's keys in shared memory; longer runs are read from the workspace

struct SelShared {
  uint32_t hist[2][kBins];
  uint32_t xch[4][8];   // what the cluster's other CTAs read, a row per exchange (16-byte aligned)
  uint32_t red[kSelThreads / 32][8];
  uint32_t scan[kSelThreads / 32];
  uint32_t at[4];
};

constexpr size_t kMostShared = sizeof(SelShared) + kMaxWords * 4 + kEvictSlots / 8 / 32 * 12;
static_assert(kMostShared <= 227 * 1024, "a CTA's shared memory");

// Sum over the CTA's threads before this one, and the sum of all. (The selection runs each
// part of its code once, so its size is time: nothing in it is unrolled without need.)
template <int NT>
SPATTEN_DEV uint2 block_scan(SelShared& sh, uint32_t x) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 31) sh.scan[warp] = y;
  __syncthreads();
  const uint32_t v = lane < NT / 32 ? sh.scan[lane] : 0u;
  return make_uint2(__reduce_add_sync(0xffffffffu, lane < warp ? v : 0u) + y - x, __reduce_add_sync(0xffffffffu, v));
}

// The lowest m bits that are set in t.
SPATTEN_DEV uint32_t lowest_bits(uint32_t t, uint32_t m) {
  while ((uint32_t)__popc(t) > m) t ^= 1u << (31 - __clz(t));
  return t;
}

// The largest cluster, whose loops over CTAs are unrolled: their loads from the
// others' shared memory go out together.
constexpr int kCluster = 8;

// CACHED: a run's keys (and positions) fit the shared memory. POOL: plan.by_pool.
template <bool CACHED, int NT, bool POOL>
__global__ void __launch_bounds__(NT) paged_select_kernel(const PagedEvictParams p, const EvictPlan plan,
                                                                   int run, int cached) {
  extern __shared__ __align__(16) uint8_t dsm[];
  SelShared& sh = *reinterpret_cast<SelShared*>(dsm);
  uint32_t* keys = reinterpret_cast<uint32_t*>(dsm + sizeof(SelShared));  // [cached]
  uint32_t* prot = keys + cached;                                          // [run / 32]: recent
  uint32_t* kept = prot + run / 32;                                        // [run / 32]
  uint32_t* ties = kept + run / 32;                                        // [run / 32]
  grid_dependents();
  grid_wait();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), CL = (int)cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.z, hl = blockIdx.y;
  const int G = p.c.G, page = p.c.page, page_log = __ffs(page) - 1, keep = p.keep;
  const int64_t line = (int64_t)b * plan.lines_per_b + hl;
  const int len = *(p.lens + b);
  uint32_t* const head = plan.head + line * 4;
  auto leave_alone = [&]() {
    if (rank == 0 && tid == 0) {
      head[0] = 0u;
      head[1] = (uint32_t)len;
    }
  };
  if (len <= keep || len > plan.usable) {  // (the same for the whole cluster)
    leave_alone();
    return;
  }
  // tables that are wider than the pool: the CTAs share the sequence's own slots (48 by head in tables
  // of ten times their slots: 151 us, 175 in runs of the table's)
  int part = run;
  if constexpr (POOL) part = min(run, (((len + CL - 1) >> (__ffs(CL) - 1)) + 31) / 32 * 32);  // (CL: 1 to 8)
  const int lo = min(rank * part, len), n = min(part, len - lo), words = (n + 31) / 32;

  auto at = [&](int i) { return POOL ? pooled_key(p.c, plan, b, hl, lo + i, page_log) : line * plan.pitch + lo + i; };
  auto key = [&](int i) { return CACHED ? keys[i] : plan.key[at(i)]; };

  // keys, the newest position, whether every slot has memory (pitch and runs are multiples of 32)
  int newest = INT_MIN;
  bool hole = false;
#pragma unroll 2
  for (int i = 4 * tid; i < n; i += 4 * NT) {
    const int64_t from = at(i);
    uint4 k = make_uint4(kNoKey, kNoKey, kNoKey, kNoKey);
    if (!POOL || from >= 0) k = *reinterpret_cast<const uint4*>(plan.key + from);
    const uint32_t x[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) hole |= i + j < n && x[j] == kNoKey;
    if (CACHED) *reinterpret_cast<uint4*>(keys + i) = k;
  }
  if (p.recent > 0) {
#pragma unroll 2
    for (int i = 4 * tid; i < n; i += 4 * NT) {
      const int64_t from = at(i);
      int4 k = make_int4(INT_MIN, INT_MIN, INT_MIN, INT_MIN);
      if (!POOL || from >= 0) k = *reinterpret_cast<const int4*>(plan.place + from);
      const int x[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < n) newest = max(newest, x[j]);
    }
  }
  {
    const int top = __reduce_max_sync(0xffffffffu, newest);
    const bool any = __any_sync(0xffffffffu, hole);
    if (lane == 0) {
      sh.red[warp][0] = (uint32_t)top;
      sh.red[warp][1] = any;
    }
    __syncthreads();
    if (warp == 0) {
      const bool in = lane < NT / 32;
      const int m = __reduce_max_sync(0xffffffffu, in ? (int)sh.red[lane][0] : INT_MIN);
      const uint32_t h = __reduce_max_sync(0xffffffffu, in ? sh.red[lane][1] : 0u);
      if (lane == 0) {
        sh.xch[0][0] = (uint32_t)m;
        sh.xch[0][1] = h;
      }
    }
    cl.sync();
    const uint2 x = lane < CL ? *reinterpret_cast<const uint2*>(cl.map_shared_rank(&sh.xch[0][0], lane))
                              : make_uint2((uint32_t)INT_MIN, 0u);
    newest = __reduce_max_sync(0xffffffffu, (int)x.x);
    const uint32_t h = __reduce_max_sync(0xffffffffu, x.y);
    if (h) {
      leave_alone();
      cl.sync();
      return;
    }
  }
  // the recent ones; how many they are, and the range of the keys of both classes
  {
    uint32_t cnt = 0u, lo0 = 0xFFFFFFFFu, hi0 = 0u, lo1 = 0xFFFFFFFFu, hi1 = 0u;
#pragma unroll 2
    for (int base = 0; base < words * 32; base += NT) {
      const int i = base + tid;
      bool r = false;
      if (i < n) {
        if (p.recent > 0) r = (int64_t)plan.place[at(i)] > (int64_t)newest - p.recent;
        const uint32_t k = key(i);
        if (r) {
          lo1 = min(lo1, k);
          hi1 = max(hi1, k);
        } else {
          lo0 = min(lo0, k);
          hi0 = max(hi0, k);
        }
      }
      const uint32_t m = __ballot_sync(0xffffffffu, r);
      if (lane == 0 && i < words * 32) {
        prot[i >> 5] = m;
        cnt += __popc(m);
      }
    }
    lo0 = __reduce_min_sync(0xffffffffu, lo0);
    hi0 = __reduce_max_sync(0xffffffffu, hi0);
    lo1 = __reduce_min_sync(0xffffffffu, lo1);
    hi1 = __reduce_max_sync(0xffffffffu, hi1);
    if (lane == 0) {
      sh.red[warp][0] = cnt;
      sh.red[warp][1] = lo0;
      sh.red[warp][2] = hi0;
      sh.red[warp][3] = lo1;
      sh.red[warp][4] = hi1;
    }
    __syncthreads();
    if (warp == 0) {
      const bool in = lane < NT / 32;
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const uint32_t v = in ? sh.red[lane][i] : (i & 1 ? 0xFFFFFFFFu : 0u);
        const uint32_t y = i == 0 ? __reduce_add_sync(0xffffffffu, v)
                                  : i & 1 ? __reduce_min_sync(0xffffffffu, v) : __reduce_max_sync(0xffffffffu, v);
        if (lane == 0) sh.xch[1][i] = y;
      }
    }
    cl.sync();
  }
  uint4 range = make_uint4(0u, 0xFFFFFFFFu, 0u, 0xFFFFFFFFu);
  uint32_t r_hi = 0u;
  if (lane < CL) {
    range = *reinterpret_cast<const uint4*>(cl.map_shared_rank(&sh.xch[1][0], lane));
    r_hi = *cl.map_shared_rank(&sh.xch[1][4], lane);
  }
  const uint32_t recents = __reduce_add_sync(0xffffffffu, range.x);
  uint32_t k_lo = __reduce_min_sync(0xffffffffu, range.y), k_hi = __reduce_max_sync(0xffffffffu, range.z);
  const bool cls = recents >= (uint32_t)keep;  // the class that is chosen from: the recent ones, or the others
  if (cls) {
    k_lo = __reduce_min_sync(0xffffffffu, range.w);
    k_hi = __reduce_max_sync(0xffffffffu, r_hi);
  }
  uint32_t need = cls ? keep : keep - recents;  // of the class; its largest keys
  // radix rounds: keys above k_hi are kept, the need-th largest lies in [k_lo, k_hi]
  bool whole = false, every = false;  // no ties: the class's keys above k_hi are kept; all of its keys are
  for (int round = 0; !whole; ++round) {
    const uint32_t span = k_hi - k_lo;
    const int shift = span < (uint32_t)kBins ? 0 : 32 - __clz(span) - 11;
    uint32_t* hist = sh.hist[round & 1];
    for (int i = tid; i < kBins; i += NT) hist[i] = 0u;
    __syncthreads();
#pragma unroll 2
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = key(i);
      if (((prot[i >> 5] >> (i & 31)) & 1u) == (uint32_t)cls && k >= k_lo && k <= k_hi) atomicAdd(&hist[(k - k_lo) >> shift], 1u);
    }
    cl.sync();
    // bins from the top: thread t takes the PER bins that end at kBins - 1 - PER t
    constexpr int PER = kBins / NT;
    uint32_t c[PER], mine = 0u;
#pragma unroll
    for (int j = 0; j < PER; ++j) c[j] = 0u;
#pragma unroll
    for (int r = 0; r < kCluster; ++r) {
      if (r >= CL) continue;
      const uint2* x = reinterpret_cast<const uint2*>(cl.map_shared_rank(hist, r) + kBins - PER - PER * tid);
#pragma unroll
      for (int j = 0; j < PER; j += 2) {
        const uint2 y = x[j / 2];
        c[PER - 1 - j] += y.x;
        c[PER - 2 - j] += y.y;
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) mine += c[j];
    uint32_t above = block_scan<NT>(sh, mine).x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (above < need && need <= above + c[j]) {
        sh.at[0] = kBins - 1 - (tid * PER + j);
        sh.at[1] = above;
        sh.at[2] = c[j];
      }
      above += c[j];
    }
    __syncthreads();
    const uint32_t bin = sh.at[0], in = sh.at[2];
    need -= sh.at[1];
    const uint32_t b_lo = k_lo + (bin << shift);
    const uint32_t b_hi = min(k_hi, b_lo + ((1u << shift) - 1u));
    __syncthreads();  // sh.at is read
    if (need == in) {  // all of the bin are kept
      whole = true;
      every = b_lo == 0u;
      k_hi = b_lo - 1u;
    } else {
      k_lo = b_lo;
      k_hi = b_hi;
      if (shift == 0) break;  // one key: `need` of those that have it
    }
  }
  // kept for sure, and the ones of the border's key
  uint32_t n_ties = 0u;
#pragma unroll 2
  for (int base = 0; base < words * 32; base += NT) {
    const int i = base + tid;
    bool sure = false, tie = false;
    if (i < n) {
      const bool mine = ((prot[i >> 5] >> (i & 31)) & 1u) == (uint32_t)cls;
      const uint32_t k = key(i);
      sure = mine ? every || k > k_hi : !cls;  // (chosen among the others: all recent ones stay)
      tie = mine && !whole && k == k_hi;
    }
    const uint32_t ms = __ballot_sync(0xffffffffu, sure), mt = __ballot_sync(0xffffffffu, tie);
    if (lane == 0 && i < words * 32) {
      kept[i >> 5] = ms;
      ties[i >> 5] = mt;
      n_ties += __popc(mt);
    }
  }
  {
    const uint32_t total = block_scan<NT>(sh, n_ties).y;
    if (tid == 0) sh.xch[2][0] = total;
    cl.sync();
  }
  const uint32_t before = __reduce_add_sync(0xffffffffu, lane < rank ? *cl.map_shared_rank(&sh.xch[2][0], lane) : 0u);
  uint32_t left = whole || before >= need ? 0u : need - before;  // ties that this CTA's slots may still keep
  uint32_t n_dst = 0u, n_src = 0u;
  for (int base = 0; base < words; base += NT) {
    const int w = base + tid;
    const uint32_t t = w < words ? ties[w] : 0u;
    const uint2 ties_at = block_scan<NT>(sh, __popc(t));
    const uint32_t at = ties_at.x;
    if (w < words) {
      const uint32_t k = kept[w] | (at < left ? lowest_bits(t, left - at) : 0u);
      kept[w] = k;
      const int s0 = lo + 32 * w;  // slots before `keep` of the word
      const uint32_t front = s0 + 32 <= keep ? 0xFFFFFFFFu : s0 >= keep ? 0u : (1u << (keep - s0)) - 1u;
      n_dst += __popc(front & ~k);
      n_src += __popc(k & ~front);
    }
    left -= min(left, ties_at.y);
  }
  {
    const uint32_t td = block_scan<NT>(sh, n_dst).y, ts = block_scan<NT>(sh, n_src).y;
    if (tid == 0) {
      sh.xch[3][0] = td;
      sh.xch[3][1] = ts;
    }
    cl.sync();
  }
  const uint2 counts = lane < CL ? *reinterpret_cast<const uint2*>(cl.map_shared_rank(&sh.xch[3][0], lane)) : make_uint2(0u, 0u);
  const uint32_t moves = __reduce_add_sync(0xffffffffu, counts.x);
  uint32_t d0 = __reduce_add_sync(0xffffffffu, lane < rank ? counts.x : 0u);
  uint32_t s0 = __reduce_add_sync(0xffffffffu, lane < rank ? counts.y : 0u);
  uint32_t base = (uint32_t)(line * plan.cap);
  if (POOL) {
    if (rank == 0 && tid == 0) {
      const unsigned long long first_place = atomicAdd(plan.used, (unsigned long long)moves);
      sh.xch[0][0] = (uint32_t)first_place;
      sh.xch[0][1] = first_place + moves <= (unsigned long long)plan.room;
    }
    cl.sync();
    const uint2 x = *reinterpret_cast<const uint2*>(cl.map_shared_rank(&sh.xch[0][0], 0));
    if (!x.y) {
      leave_alone();
      cl.sync();
      return;
    }
    base = x.x;
  }
  int32_t* const dst = plan.dst + base;
  int32_t* const src = plan.src + base;
  int32_t* const first = plan.first + line * (plan.blocks + 1);
  auto front_of = [&](int w) {  // slots before `keep` of a word
    const int at = lo + 32 * w;
    return at + 32 <= keep ? 0xFFFFFFFFu : at >= keep ? 0u : (1u << (keep - at)) - 1u;
  };
  for (int base = 0; base < words; base += NT) {  // numbers of the words' first free and moving slots
    const int w = base + tid;
    const uint32_t k = w < words ? kept[w] : 0u, front = w < words ? front_of(w) : 0u;
    const uint2 d = block_scan<NT>(sh, __popc(front & ~k)), s = block_scan<NT>(sh, __popc(k & ~front));
    if (w < words) {
      prot[w] = d0 + d.x;
      ties[w] = s0 + s.x;
    }
    d0 += d.y;
    s0 += s.y;
  }
  __syncthreads();
  for (int w = warp; w < words; w += NT / 32) {  // a slot per lane
    const int slot = lo + 32 * w + lane;
    const uint32_t k = kept[w], front = front_of(w), free = front & ~k, move = k & ~front, before_me = (1u << lane) - 1u;
    const uint32_t d = prot[w] + __popc(free & before_me);
    if ((free >> lane) & 1u) dst[d] = slot;
    if ((move >> lane) & 1u) src[ties[w] + __popc(move & before_me)] = slot;
    if (slot < keep && (slot & (page - 1)) == 0) first[slot >> page_log] = d;
  }
  if (rank == 0) {
    if (tid == 0) {
      head[0] = moves;
      head[1] = (uint32_t)keep;
      head[2] = base;
      first[plan.blocks] = (int)moves;
    }
    // the block of slot `keep` may change its scale while others read its tokens
    const int g0 = p.per_head ? hl : 0, g1 = p.per_head ? hl + 1 : G;
    for (int g = g0 + tid; g < g1; g += NT) {
      const int64_t blk = (int64_t)paged_page(p.c, b, keep >> page_log) * G + g;
      float* e = plan.edge + ((int64_t)b * G + g) * 2;
      e[0] = p.c.k_scale[blk];
      e[1] = p.c.v_scale[blk];
    }
  }
  cl.sync();  // no CTA leaves while its shared memory is read
}

// A CTA per block (page, KV head), K and V together: most of the time is the chain of
// loads plan, page, codes. (Four blocks a CTA one after the other, 256 threads: the
// 72 us above were 82.)
template <int KV, int D, int PAGE>
__global__ void __launch_bounds__(MoveShape<D, PAGE>::NT) paged_move_kernel(const PagedEvictParams p,
                                                                           const EvictPlan plan) {
  __shared__ MoveRows<PAGE> m;
  grid_dependents();
  grid_wait();
  const int b = blockIdx.z, g = blockIdx.y, G = p.c.G, tid = threadIdx.x, blk = blockIdx.x;
  const int64_t line = (int64_t)b * plan.lines_per_b + (p.per_head ? g : 0);
  const uint4 head = *reinterpret_cast<const uint4*>(plan.head + line * 4);
  if (blk == 0 && g == 0 && tid == 0) p.new_lens[b] = (int)head.y;
  if (head.x == 0) return;
  const int32_t* first = plan.first + line * (plan.blocks + 1) + blk;
  const int f0 = first[0], f1 = first[1];
  if (f1 <= f0) return;
  const int end = min(p.keep - blk * PAGE, PAGE), edge = p.keep / PAGE;
  const int64_t to = (int64_t)paged_page(p.c, b, blk) * G + g;
  if (tid < PAGE) m.src[tid] = kNoRow;
  __syncthreads();
  const float2 edge_scale = *reinterpret_cast<const float2*>(plan.edge + ((int64_t)b * G + g) * 2);
  if (f0 + tid < f1) {  // a move per thread
    const int s = plan.src[head.z + f0 + tid], d = plan.dst[head.z + f0 + tid] - blk * PAGE;
    const int64_t from = (int64_t)paged_page(p.c, b, s / PAGE) * G + g, row = from * PAGE + s % PAGE;
    m.src[d] = (uint32_t)row;
    m.scale[0][d] = s / PAGE == edge ? edge_scale.x : p.c.k_scale[from];
    m.scale[1][d] = s / PAGE == edge ? edge_scale.y : p.c.v_scale[from];
    p.weight[to * PAGE + d] = p.weight[row];
    p.position[to * PAGE + d] = p.position[row];
  }
  const float2 was = blk == edge ? edge_scale : make_float2(p.c.k_scale[to], p.c.v_scale[to]);
  __syncthreads();
  move_block<KV, D, PAGE>(m, p.c, to, was, f1 - f0 < end, end);
}

// ---------------------------------------------------------------- accepted tokens

// A CTA per (KV head, sequence) walks the blocks that accepted tokens move into, in
// order: what it reads lies at or behind what it writes. Accepted branches are short, so the
// walk is a block or two: one sequence 3.8 us, 64 5.4 us, the chain of loads.
template <int KV, int D, int PAGE>
__global__ void __launch_bounds__(MoveShape<D, PAGE>::NT) paged_keep_kernel(const PagedKeepParams p) {
  using S = MoveShape<D, PAGE>;
  __shared__ MoveRows<PAGE> m;
  __shared__ int stop, fixed;
  grid_dependents();
  grid_wait();
  const int b = blockIdx.y, g = blockIdx.x, G = p.c.G, tid = threadIdx.x;
  const PagedSeq sq = paged_seq(p.b, p.c, b);
  const int32_t* acc = p.accepted + (int64_t)b * p.accepted_st;
  // the list ends at the first entry that is not above the one before it, is no new token, or has no memory
  if (tid == 0) stop = p.A;
  __syncthreads();
  for (int j = tid; j < p.A; j += S::NT) {
    const int a = acc[j], slot = sq.old + a;
    if (a <= (j ? acc[j - 1] : -1) || a >= sq.n || slot < 0 || slot >= sq.len || paged_page(p.c, b, slot / PAGE) < 0)
      atomicMin(&stop, j);
  }
  __syncthreads();
  const int count = stop;
  if (blockIdx.x == 0 && tid == 0) p.new_lens[b] = sq.n == 0 ? *(p.b.lens + b) : max(sq.old + count, 0);
  if (tid == 0) fixed = count;
  __syncthreads();
  for (int j = tid; j < count; j += S::NT)
    if (acc[j] != j) atomicMin(&fixed, j);
  __syncthreads();
  if (fixed >= count) return;
  const int slot0 = sq.old + fixed, slot1 = sq.old + count;  // slots that tokens move into
  for (int blk = slot0 / PAGE; blk * PAGE < slot1; ++blk) {
    const int lo = max(slot0 - blk * PAGE, 0), hi = min(slot1 - blk * PAGE, PAGE);
    const int pid = paged_page(p.c, b, blk);
    if (pid < 0) continue;  // (no page here: nothing to write to)
    const int64_t to = (int64_t)pid * G + g;
    for (int r = tid; r < PAGE; r += S::NT) {
      m.src[r] = kNoRow;
      if (r >= lo && r < hi) {
        const int s = sq.old + acc[blk * PAGE + r - sq.old];
        const int64_t from = (int64_t)paged_page(p.c, b, s / PAGE) * G + g, row = from * PAGE + s % PAGE;
        m.src[r] = (uint32_t)row;
        m.scale[0][r] = p.c.k_scale[from];
        m.scale[1][r] = p.c.v_scale[from];
      }
    }
    const float2 was = make_float2(p.c.k_scale[to], p.c.v_scale[to]);
    __syncthreads();
    if (p.weight) {  // a row per thread, read before any is written
      const int r = lo + tid;
      const float w = r < hi ? p.weight[m.src[r]] : 0.f;
      const int x = r < hi ? p.position[m.src[r]] : 0;
      __syncthreads();
      if (r < hi) {
        p.weight[to * PAGE + r] = w;
        p.position[to * PAGE + r] = x;
      }
    }
    move_block<KV, D, PAGE>(m, p.c, to, was, lo > 0, lo);
    __syncthreads();  // the block is written, its list read
  }
}

// Slots that a sequence may hold: those of its table, and no more than the pool has.
int64_t usable_slots(const PagedEvictParams& p) {
  return (int64_t)(p.c.max_pages < p.c.P ? p.c.max_pages : p.c.P) * p.c.page;
}

struct EvictSplit {
  int cluster, run, cached, threads;
  size_t smem;
};

EvictSplit split_for(const PagedEvictParams& p, int n_sm) {
  const int64_t slots = usable_slots(p);
  EvictSplit s;
  const int64_t lines = (int64_t)p.B * (p.per_head ? p.c.G : 1);
  s.cluster = 1;
  while (s.cluster < kCluster && slots > (int64_t)s.cluster * (lines * s.cluster < n_sm ? 2048 : 16384)) s.cluster *= 2;
  s.run = (int)((slots + s.cluster - 1) / s.cluster + 31) / 32 * 32;
  s.cached = s.run <= kMaxWords ? s.run : 0;
  s.threads = lines * s.cluster > n_sm && s.run <= 16384 ? 512 : 1024;
  s.smem = sizeof(SelShared) + (size_t)s.cached * 4 + (size_t)s.run / 32 * 12;
  return s;
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// plan (pointers null) and bytes
size_t plan_for(const PagedEvictParams& p, void* ws, EvictPlan& x) {
  const int64_t slots = usable_slots(p), pool = (int64_t)p.c.P * p.c.page;
  x.usable = (int)slots;
  x.by_pool = pool < (int64_t)p.B * p.c.max_pages * p.c.page;
  x.lines_per_b = p.per_head ? p.c.G : 1;
  const int64_t kept = p.keep < slots ? p.keep : slots;
  x.blocks = (int)((kept + p.c.page - 1) / p.c.page);
  x.cap = (int)(kept < slots - kept ? kept : slots - kept);
  const size_t lines = (size_t)p.B * x.lines_per_b;
  uint8_t* w = static_cast<uint8_t*>(ws);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* r = w + at;
    at += align256(bytes);
    return w ? r : nullptr;
  };
  x.head = reinterpret_cast<uint32_t*>(take(lines * 16));
  x.used = reinterpret_cast<unsigned long long*>(take(8));
  x.first = reinterpret_cast<int32_t*>(take(lines * (x.blocks + 1) * 4));
  x.room = (int64_t)lines * x.cap;  // (fewer than 2^32: the pool has fewer rows)
  if (x.by_pool && x.room > x.lines_per_b * pool) x.room = x.lines_per_b * pool;
  x.dst = reinterpret_cast<int32_t*>(take(x.room * 4));
  x.src = reinterpret_cast<int32_t*>(take(x.room * 4));
  x.edge = reinterpret_cast<float*>(take((size_t)p.B * p.c.G * 8));
  x.pitch = (int)((slots + 31) / 32 * 32);
  const size_t keys = (x.by_pool ? (size_t)x.lines_per_b * pool : lines * x.pitch) * 4;
  x.key = reinterpret_cast<uint32_t*>(take(keys));
  x.place = reinterpret_cast<int32_t*>(take(p.recent > 0 ? keys : 0));
  return at;
}

template <int KV, int D, int PAGE>
cudaError_t move_launch(const PagedEvictParams& p, const EvictPlan& plan, cudaStream_t st) {
  return launch_dependent(paged_move_kernel<KV, D, PAGE>,
                          dim3(plan.blocks, p.c.G, p.B), MoveShape<D, PAGE>::NT, 0, st, p, plan);
}
template <int KV, int D, int PAGE>
cudaError_t keep_launch(const PagedKeepParams& p, cudaStream_t st) {
  return launch_dependent(paged_keep_kernel<KV, D, PAGE>, dim3(p.c.G, p.b.B), MoveShape<D, PAGE>::NT, 0, st, p);
}

// f(KV, D, PAGE) as constants
template <typename F>
cudaError_t with_shape(int kv, int D, int page, F f) {
  auto pages = [&](auto k, auto d) {
    switch (page) {
      case 16: return f(k, d, std::integral_constant<int, 16>{});
      case 32: return f(k, d, std::integral_constant<int, 32>{});
      case 64: return f(k, d, std::integral_constant<int, 64>{});
      case 128: return f(k, d, std::integral_constant<int, 128>{});
      default: return cudaErrorInvalidValue;
    }
  };
  auto dims = [&](auto k) {
    if (D == 128) return pages(k, std::integral_constant<int, 128>{});
    if (D == 64) return pages(k, std::integral_constant<int, 64>{});
    return cudaErrorInvalidValue;
  };
  return kv == kKvInt8 ? dims(std::integral_constant<int, kKvInt8>{}) : dims(std::integral_constant<int, kKvE4m3>{});
}

template <bool CACHED, int NT, bool POOL>
cudaError_t select_launch_as(const PagedEvictParams& p, const EvictPlan& plan, const EvictSplit& s, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may use its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
    e = cudaFuncSetAttribute(paged_select_kernel<CACHED, NT, POOL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)kMostShared);
    if (e != cudaSuccess) return e;
    if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(s.cluster, plan.lines_per_b, p.B);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = s.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, paged_select_kernel<CACHED, NT, POOL>, p, plan, s.run, s.cached);
}

template <bool CACHED, int NT>
cudaError_t select_launch(const PagedEvictParams& p, const EvictPlan& plan, const EvictSplit& s, cudaStream_t st) {
  return plan.by_pool ? select_launch_as<CACHED, NT, true>(p, plan, s, st)
                      : select_launch_as<CACHED, NT, false>(p, plan, s, st);
}

}  // namespace

size_t paged_evict_workspace(const PagedEvictParams& p) {
  EvictPlan x;
  return plan_for(p, nullptr, x);
}

cudaError_t launch_paged_evict(const PagedEvictParams& p, int kv, void* ws, int n_sm, cudaStream_t st) {
  EvictPlan plan;
  plan_for(p, ws, plan);
  const dim3 slots((unsigned)((plan.pitch + kRankSlots - 1) / kRankSlots), plan.lines_per_b, p.B);
  cudaError_t e = launch_dependent(paged_rank_kernel, slots, kRankThreads, 0, st, p, plan);
  if (e != cudaSuccess) return e;
  const EvictSplit s = split_for(p, n_sm);
  if (s.cached == 0) e = select_launch<false, 1024>(p, plan, s, st);
  else e = s.threads == 1024 ? select_launch<true, 1024>(p, plan, s, st) : select_launch<true, 512>(p, plan, s, st);
  if (e != cudaSuccess) return e;
  return with_shape(kv, p.c.D, p.c.page, [&](auto k, auto d, auto page) {
    return move_launch<decltype(k)::value, decltype(d)::value, decltype(page)::value>(p, plan, st);
  });
}

cudaError_t launch_paged_keep(const PagedKeepParams& p, int kv, cudaStream_t st) {
  return with_shape(kv, p.c.D, p.c.page, [&](auto k, auto d, auto page) {
    return keep_launch<decltype(k)::value, decltype(d)::value, decltype(page)::value>(p, st);
  });
}

}  // namespace spatten
