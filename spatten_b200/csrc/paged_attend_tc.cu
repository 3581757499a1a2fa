// Attention over the paged 8-bit KV cache for many query rows per KV head
// (pieces of prompts): the tcgen05 path of spatten_paged_attend.
//
// The R = H / G query heads of a KV head and the n new tokens of a sequence are
// n R query rows over the same keys. A CTA takes 256 of them (two row tiles of
// 128) and walks key tiles of 64:
//   S [128 x 64] = Q' . K codes^T,  O [128 x D] += W . V codes   (kind::f16)
// with f16 operands (every int8 and e4m3 code is an f16; q' = q 2^e, see
// query_scale) and fp32 accumulators in tensor memory. One thread owns a
// query row:
//   t = S (sm_scale log2(e) 2^-e k_scale),  w = 2^(t + log2 v_scale - M),
// with a reference M that follows max(t + log2 v_scale), kRoom below it, so that W
// keeps 11 bits whatever the blocks' scales are; O is rescaled in tensor memory when
// that maximum grew by more than kSlack. The softmax's sum l needs p = 2^(t - m): within a block w
// and p differ by the factor 2^(M - log2 v_scale - m), so l takes the block's sum
// of w times it (one exponential per score), except where w could underflow
// under it, which takes the exponentials of p.
//
// 20 warps, one CTA per SM:
//   warps 0-3, 4-7  softmax of the two row tiles: S from tensor memory, W into the
//                   columns that S came from, rescaling, the epilogue and the next
//                   queries;
//   warps 8-15      codes to f16: 16-byte loads a tile ahead, widened into a
//                   ring of K / V tiles in the layouts that the MMAs read (K
//                   K-major, V MN-major: both [64-dim block][key][128 B]);
//   warps 16-19     MMA issue, one thread each: S and O of the two row tiles (one
//                   thread for all took 3600 of a tile's 4450 cycles).
// A tile's codes are widened once for 256 rows, and two row tiles keep the
// tensor cores busy through each other's softmax. S has two buffers per row tile, so
// that the next S and the product with W run under a tile's exponentials; with W
// in one shared-memory buffer a tile's exponentials had to wait for the product of
// the tile before (512 new tokens over 32768: 376 us instead of 320).
//
// 512 new tokens over 32768 (32 heads, 8 KV heads, D = 128, int8): 320 us, 854
// TFLOP/s, 0.51 of the measured bf16 rate; 1024 over 8192, 2 sequences, e4m3: 343 us,
// 752 TFLOP/s; a prompt of 4096: 223 us, 616 TFLOP/s. What bounds it: one thread per
// row takes a tile's 64 scores through a chain of load, maximum, exponentials and
// store that two warps per scheduler do not hide; then a line's set-up (queries,
// the first tile, the epilogue).
//
// Work split: as in paged_attend.cu, ranges of equal length over all CTAs, here in
// keys: row tile rt of a sequence counts old + (rt + 1) 256 / R of them (the causal
// triangle) and kLineCost, cumulated in closed form, and the 64-key tile at
// position k belongs to the CTA that holds unit kLineCost + k of its line. Every
// wait is bounded; a timeout records a code in this file's device error word and
// the CTA winds down.
#include <atomic>
#include <cmath>

#include "kernels.h"
#include "paged_dev.cuh"
#include "paged_join.cuh"
#include "sm100.cuh"

namespace spatten {
namespace {

using namespace sm100;

constexpr int kRowTile = 128, kRowsCta = 256, kKeys = 64, kRing = 4;
constexpr int kSoftWarps = 8, kWideWarps = 8, kMmaWarps = 4,
              kThreads = 32 * (kSoftWarps + kWideWarps + kMmaWarps);
// registers per thread at launch, and of each role after setmaxnreg
constexpr int kRegs = 96, kSoftRegs = 152, kWideRegs = 64, kMmaRegs = 48;
static_assert(kSoftWarps * kSoftRegs + kWideWarps * kWideRegs + kMmaWarps * kMmaRegs ==
                  (kSoftWarps + kWideWarps + kMmaWarps) * kRegs,
              "the roles share what the block was launched with");
// What a line's set-up takes, in keys: the queries, the first tile's way through
// the pipeline and the epilogue, about 10 us at 1.2 us per 64-key tile. Measured on
// a prompt of 4096 tokens and a piece of 862 over 7000: 256 keys 268 and 150 us,
// 512 222 and 152 us, 896 229 and 160 us.
constexpr uint32_t kLineCost = 512;
constexpr unsigned kErr = 0x400;
constexpr int kMaxBatch = 1024;

template <int D>
struct Lay {
  static constexpr int kTileBytes = kKeys * D * 2;       // K or V, f16
  static constexpr int kQBytes = kRowTile * D * 2;
  static constexpr int oQ = 0;                            // [2][D / 64][128][128 B]
  static constexpr int oKV = oQ + 2 * kQBytes;            // [ring][K | V][D / 64][64][128 B]
  static constexpr int oScale = oKV + kRing * 2 * kTileBytes;  // [ring][ks 4, log2 vs 4, have]
  static constexpr int kScaleStride = 48;
  static constexpr int oBar = oScale + kRing * kScaleStride;
  static constexpr int kNumBars = 2 * kRing + 4 + 4 + 4 + 2 + 4;
  static constexpr int oTmem = oBar + kNumBars * 8;
  static constexpr int oAbort = oTmem + 4;
  static constexpr int oScan = (oAbort + 4 + 7) & ~7;     // [32] 64-bit
  static constexpr int oPre = oScan + 256;                // [B + 1]
  static constexpr int bytes(int B) { return oPre + (B + 1) * 4 + 1024; }
};

SPATTEN_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
SPATTEN_DEV void tmem_st32f(uint32_t taddr, const float* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
      "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]),
      "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]),
      "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31]));
}
SPATTEN_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Four codes in order as two f16 pairs.
template <int KV>
SPATTEN_DEV uint2 widen4(uint32_t w) {
  if constexpr (KV == kKvInt8) {
    const uint32_t x = w ^ 0x80808080u;  // byte u under 0x64 is the f16 1024 + u = 1152 + code
    uint32_t lo = __byte_perm(x, 0x64646464u, 0x4140), hi = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 b = __half2half2(__ushort_as_half(0x6480));
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), b);
    const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&hi), b);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
  } else {
    return make_uint2(e4m3x2_to_f16x2(w & 0xFFFFu), e4m3x2_to_f16x2(w >> 16));
  }
}

// A CTA's run of units, as segments of lines. Every role walks it by itself.
struct Segments {
  const PagedAttendParams& p;
  const uint32_t* pre;
  uint32_t u, u1;
  int b, R;
  // the current segment
  PagedSeq sq;
  int g, r0, nrows, lim_max, t0, t1;
  bool first, whole;     // begins the line; is all of it
  uint32_t u0, line;     // the segment's first unit; units of the line

  SPATTEN_DEV static uint32_t tokens_per_tile(int R) { return (kRowsCta + R - 1) / R; }
  // units of row tiles 0 .. rt - 1 of a sequence (`old` within the page table)
  template <typename U = uint32_t>
  SPATTEN_DEV static U before(const PagedAttendParams& p, const PagedSeq& s, uint32_t rt, uint32_t tok) {
    const uint32_t old = min(max(s.old, 0), p.c.max_pages * p.c.page);
    return U(rt) * (old + kLineCost) + tok * (U(rt) * (rt + 1) / 2);
  }
  SPATTEN_DEV static uint32_t row_tiles(const PagedSeq& s, int R) { return ((uint32_t)s.n * R + kRowsCta - 1) / kRowsCta; }
  SPATTEN_DEV static unsigned long long units(const PagedAttendParams& p, const PagedSeq& s, int R) {
    return before<unsigned long long>(p, s, row_tiles(s, R), tokens_per_tile(R));
  }

  SPATTEN_DEV bool next() {
    if (u >= u1) return false;
    while (pre[b + 1] <= u) ++b;
    sq = paged_seq(p.b, p.c, b);
    const uint32_t tok = tokens_per_tile(R), per = before(p, sq, row_tiles(sq, R), tok), local = u - pre[b];
    g = local / per;
    const uint32_t r = local % per;
    uint32_t lo = 0, hi = row_tiles(sq, R);  // the row tile of unit r
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) >> 1;
      if (before(p, sq, mid, tok) <= r) lo = mid; else hi = mid;
    }
    const uint32_t v0 = r - before(p, sq, lo, tok);
    u0 = u;
    line = before(p, sq, lo + 1, tok) - before(p, sq, lo, tok);
    const uint32_t v1 = min(line, v0 + (u1 - u));
    auto tile = [](uint32_t v) { return (int)((max(v, kLineCost) - kLineCost + kKeys - 1) / kKeys); };
    first = v0 == 0;
    whole = first && v1 == line;
    r0 = lo * kRowsCta;
    nrows = sq.n * R;
    lim_max = max(min(sq.old + min((r0 + kRowsCta - 1) / R, sq.n - 1) + 1, sq.len), 0);
    const int kt = (lim_max + kKeys - 1) / kKeys;
    t0 = min(tile(v0), kt);
    t1 = v1 == line ? kt : min(tile(v1), kt);
    u += v1 - v0;
    return true;
  }
};

template <int KV, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_attend_tc_kernel(const PagedAttendParams p, const PagedPartials ws,
                                                                      const bool bf16) {
  using L = Lay<D>;
  extern __shared__ uint8_t smem_raw[];
  grid_dependents();
  grid_wait();
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t bars = smem_u32(sm + L::oBar);
  const SBarArr kv_full{bars}, kv_empty{bars + 8 * kRing}, s_full{bars + 16 * kRing}, s_empty{bars + 16 * kRing + 32},
      w_full{bars + 16 * kRing + 64}, q_full{bars + 16 * kRing + 96},
      drain{bars + 16 * kRing + 112};
  volatile int* abort = reinterpret_cast<volatile int*>(sm + L::oAbort);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + L::oTmem);
  uint32_t* pre = reinterpret_cast<uint32_t*>(sm + L::oPre);
  unsigned long long* scan = reinterpret_cast<unsigned long long*>(sm + L::oScan);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = p.c.G, R = p.b.H / G;

  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(kv_full[i], kWideWarps);
      mbar_init(kv_empty[i], 2);  // the two row tiles
    }
    for (int i = 0; i < 4; ++i) {  // [row tile][buffer]
      mbar_init(s_full[i], 1);
      mbar_init(w_full[i], 4);
      mbar_init(s_empty[i], 1);  // the product with W, which lies in S's columns, is done
    }
    for (int i = 0; i < 2; ++i) mbar_init(q_full[i], 4);
    for (int i = 0; i < kMmaWarps; ++i) mbar_init(drain[i], 1);
    fence_barrier_init();
    *abort = 0;
    pre[0] = 0;
  }
  if (warp == kSoftWarps + kWideWarps) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  // prefix sums of the sequences' units. The host made sure of 32 bits
  // for sequences that share no rows; others may need more, and then nothing is done.
  unsigned long long U64 = 0;
  for (int base = 0; base < p.b.B; base += kThreads) {
    const int b = base + tid;
    unsigned long long x = 0;
    if (b < p.b.B) {
      const PagedSeq s = paged_seq(p.b, p.c, b);
      if (paged_serves(p, s, R)) x = (unsigned long long)G * Segments::units(p, s, R);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    unsigned long long front = U64;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) front += scan[w];
      U64 += scan[w];
    }
    if (b < p.b.B) pre[b + 1] = (uint32_t)(front + x);
    __syncthreads();
  }
  const uint32_t U = U64 >> 32 ? 0 : (uint32_t)U64;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  const uint32_t cta = blockIdx.x, ctas = max(min(gridDim.x, (U + kKeys - 1) / kKeys), 1u);
  const uint32_t per = U / ctas, more = U % ctas;
  Segments seg{p, pre};
  seg.R = R;
  seg.b = 0;
  seg.u = seg.u1 = 0;
  if (cta < ctas) {
    seg.u = cta * per + min(cta, more);
    seg.u1 = seg.u + per + (cta < more ? 1 : 0);
  }

  if (warp < kSoftWarps) {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs) : "memory");
    const int rt = warp >> 2, row = tid & 127;  // row tile, row in it = tensor-memory lane
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = tl + rt * 2 * kKeys, to = tl + 4 * kKeys + rt * D;
    PagedCut cut = {};
    uint32_t c = 0, kv = 0;  // tiles of this row tile, tiles of the ring
    bool alive = true;
    while (seg.next()) {
      const int r = seg.r0 + rt * kRowTile + row;
      const bool live = r < seg.nrows, used = seg.nrows - seg.r0 > rt * kRowTile;
      const int nt = seg.t1 - seg.t0, i = (live ? r : 0) / R, h = seg.g * R + (live ? r : 0) % R;
      float cq = 0.f;  // what a score of this row has to be multiplied by
      if (used && nt > 0) {
        // the warp's 32 rows, LQ lanes a row (16 bytes each), all loads in flight at once
        constexpr int LQ = D / 8, RQ = 32 / LQ;
        const int li = lane % LQ, in = lane / LQ, first = rt * kRowTile + (warp & 3) * 32;
        auto pair = [&](uint32_t w) {
          return bf16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u))
                      : __half22float2(*reinterpret_cast<const __half2*>(&w));
        };
        uint4 x[LQ];
#pragma unroll
        for (int k = 0; k < LQ; ++k) {
          const int y = seg.r0 + first + k * RQ + in;
          const uint16_t* qp = static_cast<const uint16_t*>(p.q) + 8 * li;
          x[k] = make_uint4(0u, 0u, 0u, 0u);
          if (y < seg.nrows)
            x[k] = *reinterpret_cast<const uint4*>(qp + (int64_t)(seg.sq.begin + y / R) * p.q_st +
                                                   (int64_t)(seg.g * R + y % R) * p.q_sh);
        }
#pragma unroll
        for (int k = 0; k < LQ; ++k) {
          const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
          float top = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = pair(w[j]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            if (!(f.x == f.x && f.y == f.y)) top = INFINITY;
          }
#pragma unroll
          for (int d = LQ / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          const QueryScale qs = query_scale(top, p.scale_log2);
          const float mine = __shfl_sync(0xffffffffu, qs.factor, (lane % RQ) * LQ);
          if (lane / RQ == k) cq = mine;  // this thread's row is among the step's
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = pair(w[j]);
            o[j] = pack2<__half>(f.x * qs.up, f.y * qs.up);
          }
          const int y = (warp & 3) * 32 + k * RQ + in;
          *reinterpret_cast<uint4*>(sm + L::oQ + rt * L::kQBytes + (li >> 3) * (kRowTile * 128) + y * 128 +
                                    (((li & 7) ^ (y & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        mbar_arrive_elect(q_full[rt]);
      }
      const int lim = live ? min(seg.sq.old + i + 1, seg.sq.len) : 0;
      float m = -INFINITY, M = -INFINITY, l = 0.f;
      if (!used) kv += max(nt, 0);
      for (int t = seg.t0; used && t < seg.t1; ++t, ++kv) {
        const int st = kv % kRing, buf = c & 1;
        bool ok = mbar_wait(s_full[2 * rt + buf], (c >> 1) & 1, kErr | 1, abort);
        ok = ok && mbar_wait(kv_full[st], (kv / kRing) & 1, kErr | 2, abort);  // (long complete) the tile's scales
        if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
        tc_fence_after();
        float s[kKeys];
        tmem_ld32f(ts + buf * kKeys, s);
        tmem_ld32f(ts + buf * kKeys + 32, s + 32);
        tmem_wait_ld();
        const float4 ks = *reinterpret_cast<const float4*>(sm + L::oScale + st * L::kScaleStride);
        const float4 lv4 = *reinterpret_cast<const float4*>(sm + L::oScale + st * L::kScaleStride + 16);
        const uint32_t have = *reinterpret_cast<const uint32_t*>(sm + L::oScale + st * L::kScaleStride + 32);
        float a[4] = {cq * ks.x, cq * ks.y, cq * ks.z, cq * ks.w};
        const float lv[4] = {lv4.x, lv4.y, lv4.z, lv4.w};
        const int key0 = t * kKeys;
        const bool odd = key0 + kKeys > lim || have != 15u || !(fminf(fminf(a[0], a[1]), fminf(a[2], a[3])) >= 0.f);
        if (__builtin_expect(__any_sync(0xffffffffu, odd), 0)) {  // masked keys, factors below 0 or NaN: t itself
#pragma unroll
          for (int k = 0; k < kKeys; ++k) {
            s[k] *= a[k >> 4];
            if (key0 + k >= lim || !((have >> (k >> 4)) & 1u)) s[k] = -INFINITY;
          }
          a[0] = a[1] = a[2] = a[3] = 1.f;
        }
        float top = -INFINITY, topw = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float x = s[16 * q], y = s[16 * q + 1];
#pragma unroll
          for (int k = 2; k < 16; k += 2) {
            x = fmaxf(x, s[16 * q + k]);
            y = fmaxf(y, s[16 * q + k + 1]);
          }
          x = fmaxf(x, y) * a[q];
          top = fmaxf(top, x);
          topw = fmaxf(topw, x + lv[q]);
        }
        const bool up = top > m + kSlack || topw > M + (kRoom + kSlack);
        const float Mn = up ? fmaxf(M, topw - kRoom) : M, mn = up ? fmaxf(m, top) : m;
        const float Mf = finite_or_0(Mn), mf = finite_or_0(mn);
        if (up) l *= fast_exp2(m - mf);
        const float fo = up ? fast_exp2(M - Mf) : 1.f;
        m = mn;
        M = Mn;
        float e[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) e[q] = Mf - lv[q] - mf;
        const bool wide = fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])) > 90.f;
        if (__builtin_expect(__any_sync(0xffffffffu, wide || fo != 1.f), 0)) {
          if (__any_sync(0xffffffffu, wide)) {  // w underflows where p does not: the sum of p itself
#pragma unroll
            for (int k = 0; k < kKeys; ++k) {
              const float x = fast_exp2(fmaf(s[k], a[k >> 4], -mf));
              l += e[k >> 4] > 90.f ? x : 0.f;
            }
          }
          if (t > seg.t0) {  // O is at rest once the product of the tile before is done
            ok = mbar_wait(s_empty[2 * rt + (buf ^ 1)], ((c - 1) >> 1) & 1, kErr | 3, abort);
            if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {
              float o[32];
              tmem_ld32f(to + 32 * k, o);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] *= fo;
              tmem_st32f(to + 32 * k, o);
            }
            tmem_wait_st();
          }
        }
        uint32_t w[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 a2 = make_float2(a[q], a[q]), b2 = make_float2(lv[q] - Mf, lv[q] - Mf);
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int at = 16 * q + 8 * h + 2 * k;
              float2 x = __ffma2_rn(make_float2(s[at], s[at + 1]), a2, b2);
              x.x = fast_exp2(x.x);
              x.y = fast_exp2(x.y);
              sum = __fadd2_rn(sum, x);
              w[8 * (q & 1) + 4 * h + k] = pack2<__half>(x.x, x.y);
            }
          }
          if (q & 1) tmem_st16(ts + buf * kKeys + 8 * (q - 1), w);
          l += e[q] > 90.f ? 0.f : (sum.x + sum.y) * fast_exp2(e[q]);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_elect(w_full[2 * rt + buf]);
        ++c;
      }
      // epilogue: the row's O
      if (used && nt > 0 && alive) {
        const bool ok = mbar_wait(s_empty[2 * rt + ((c - 1) & 1)], ((c - 1) >> 1) & 1, kErr | 4, abort);
        if (!__all_sync(0xffffffffu, ok)) alive = false;
        tc_fence_after();
      }
      if (!alive) break;
      if (used) {
        const float inv = seg.whole ? paged_normaliser(m, l, M) : 1.f;
        const uint32_t slot = 2 * cta + (seg.first ? 1 : 0);
        uint16_t* op = static_cast<uint16_t*>(p.out) + (int64_t)(seg.sq.begin + i) * p.o_st + (int64_t)h * p.o_sh;
#pragma unroll 1
        for (int k = 0; k < D / 32; ++k) {
          float o[32];
          __syncwarp();
          if (nt > 0) {
            tmem_ld32f(to + 32 * k, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0.f;
          }
          if (!live) continue;
          if (seg.whole) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              uint32_t x[4];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                x[q] = bf16 ? pack2<__nv_bfloat16>(o[j + 2 * q] * inv, o[j + 2 * q + 1] * inv)
                            : pack2<__half>(o[j + 2 * q] * inv, o[j + 2 * q + 1] * inv);
              *reinterpret_cast<uint4*>(op + 32 * k + j) = make_uint4(x[0], x[1], x[2], x[3]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              reinterpret_cast<float4*>(ws.o)[((size_t)slot * (D / 4) + 8 * k + j / 4) * kRowsCta + rt * kRowTile + row] =
                  make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
        }
        if (live && !seg.whole) ws.ml[slot * kRowsCta + rt * kRowTile + row] = make_float4(m, l, M, 0.f);
        tc_fence_before();
      }
      if (seg.first && !seg.whole) {  // the CTAs up to that of the line's last unit hold a part each
        const uint32_t last = seg.u0 + seg.line - 1, big = more * (per + 1);
        cut.parts = (int)(last < big ? last / (per + 1) : more + (last - big) / per) - (int)cta + 1;
        cut.row0 = seg.r0; cut.nrows = seg.nrows; cut.begin = seg.sq.begin; cut.g = seg.g;
      }
    }
    if (tid == 0) ws.cut[cta] = cut;
  } else if (warp < kSoftWarps + kWideWarps) {
    // ------------------------------------------------------------ codes to f16
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideRegs) : "memory");
    constexpr int CH = D / 16, NC = D / 64, RPI = 32 * kWideWarps / CH;  // chunks per key, chunks per thread of K (and V), keys per step
    // eight lanes of a store hold four 16-dim columns of two neighbouring keys: eight banks' worth
    const int w = tid - 32 * kSoftWarps;
    const int col = CH == 8 ? (w & 3) + ((w >> 1) & 4) : w & 3;
    const int key = CH == 8 ? ((w >> 2) & 1) + 2 * (w >> 4) : w >> 2;
    const int page_log = __ffs(p.c.page) - 1;
    int t = 0;
    bool more_tiles = true;
    int pid[NC], pid_s = -1;  // pages of this thread's keys, and of block w & 3, of the tile to load next
    auto pages = [&]() {
      auto page_of = [&](int slot) { return slot < seg.lim_max ? paged_page(p.c, seg.b, slot >> page_log) : -1; };
#pragma unroll
      for (int i = 0; i < NC; ++i) pid[i] = page_of(t * kKeys + key + RPI * i);
      pid_s = page_of(t * kKeys + 16 * (w & 3));
    };
    auto advance = [&]() {
      ++t;
      while (more_tiles && t >= seg.t1) {
        more_tiles = seg.next();
        t = seg.t0;
      }
      if (more_tiles) pages();
    };
    struct Hold {
      uint4 k[NC], v[NC];
      float ks, vs;
      uint32_t have;
      bool valid;
    };
    auto load = [&](Hold& x) {
      x.valid = more_tiles;
      if (!more_tiles) return;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int slot = t * kKeys + key + RPI * i;
        const int64_t at =
            (((int64_t)max(pid[i], 0) * G + seg.g) * p.c.page + (slot & (p.c.page - 1))) * D + col * 16;
        x.k[i] = x.v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (pid[i] >= 0) x.k[i] = *reinterpret_cast<const uint4*>(p.c.k + at);
        if (pid[i] >= 0 && slot < seg.lim_max) x.v[i] = *reinterpret_cast<const uint4*>(p.c.v + at);
      }
      x.ks = x.vs = 0.f;
      if (w < 4 && pid_s >= 0) {
        const int64_t blk = (int64_t)pid_s * G + seg.g;
        x.ks = p.c.k_scale[blk];
        x.vs = p.c.v_scale[blk];
      }
      x.have = __ballot_sync(0xffffffffu, pid_s >= 0) & 15u;
      advance();
    };
    uint32_t n = 0;
    auto store = [&](const Hold& x) {
      const int st = n % kRing;
      const bool ok = mbar_wait(kv_empty[st], ((n / kRing) & 1) ^ 1, kErr | 5, abort);
      if (!__all_sync(0xffffffffu, ok)) return false;
      uint8_t* kd = sm + L::oKV + st * 2 * L::kTileBytes + (col >> 2) * (kKeys * 128);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int row = key + RPI * i;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const uint4 c = v ? x.v[i] : x.k[i];
          const uint2 a = widen4<KV>(c.x), b = widen4<KV>(c.y), d = widen4<KV>(c.z), e = widen4<KV>(c.w);
          uint8_t* dst = kd + v * L::kTileBytes + row * 128;
          const int sub = (col & 3) * 2;
          *reinterpret_cast<uint4*>(dst + ((sub ^ (row & 7)) << 4)) = make_uint4(a.x, a.y, b.x, b.y);
          *reinterpret_cast<uint4*>(dst + (((sub + 1) ^ (row & 7)) << 4)) = make_uint4(d.x, d.y, e.x, e.y);
        }
      }
      if (w < 4) {
        float* sc = reinterpret_cast<float*>(sm + L::oScale + st * L::kScaleStride);
        sc[w] = x.ks;
        sc[4 + w] = x.vs > 0.f ? fmaxf(log2f(x.vs), kNoScale) : kNoScale;
        if (w == 0) reinterpret_cast<uint32_t*>(sc)[8] = x.have;
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_elect(kv_full[st]);
      ++n;
      return true;
    };
    t = -1;
    seg.t1 = 0;  // before the first segment
    advance();
    Hold x;
    load(x);
    while (x.valid && store(x)) load(x);
  } else {
    // ------------------------------------------------------------ MMA issue
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs) : "memory");
    if (lane == 0) {
    const int rt = (warp - kSoftWarps - kWideWarps) & 1;
    const bool scores = warp < kSoftWarps + kWideWarps + 2;
    uint32_t n = 0, c = 0, nq = 0;  // tiles of the ring, tiles and queries of this row tile
    bool ok = true;
    if (scores) {  // S = Q' K^T
      constexpr uint32_t idesc = instr_desc(1, 0, 0, 0, kRowTile, kKeys);
      const uint64_t q = smem_desc_sw128(smem_u32(sm + L::oQ + rt * L::kQBytes), 16, 1024);
      while (ok && seg.next()) {
        const int nt = seg.t1 - seg.t0;
        if (nt <= 0) continue;
        if (seg.nrows - seg.r0 <= rt * kRowTile) {
          // not in use: this thread lets the ring go for its row tile, tile by tile (a wait for a phase
          // further on would take an earlier one of the same parity for it)
          for (int j = 0; j < nt && ok; ++j, ++n) {
            ok = mbar_wait(kv_full[n % kRing], (n / kRing) & 1, kErr | 7, abort);
            if (ok) mbar_arrive(kv_empty[n % kRing]);
          }
          continue;
        }
        ok = mbar_wait(q_full[rt], nq++ & 1, kErr | 6, abort);
        for (int j = 0; j < nt && ok; ++j, ++n, ++c) {
          const uint32_t st = n % kRing, buf = c & 1;
          ok = mbar_wait(s_empty[2 * rt + buf], ((c >> 1) & 1) ^ 1, kErr | 8, abort) &&
               mbar_wait(kv_full[st], (n / kRing) & 1, kErr | 7, abort);
          if (!ok) break;
          tc_fence_after();
          const uint64_t k = smem_desc_sw128(smem_u32(sm + L::oKV + st * 2 * L::kTileBytes), 16, 1024);
          const uint32_t d = tmem + (2 * rt + buf) * kKeys;
#pragma unroll
          for (int i = 0; i < D / 16; ++i)  // the descriptors' addresses count 16 bytes
            mma_f16(d, q + (((i >> 2) * (kRowTile * 128) + (i & 3) * 32) >> 4),
                    k + (((i >> 2) * (kKeys * 128) + (i & 3) * 32) >> 4), idesc, i > 0);
          mma_commit(s_full[2 * rt + buf]);
        }
      }
    } else {  // O += W V
      constexpr uint32_t idesc = instr_desc(1, 0, 0, 1, kRowTile, D);
      const uint32_t d = tmem + 4 * kKeys + rt * D;
      while (ok && seg.next()) {
        const int nt = seg.t1 - seg.t0;
        if (seg.nrows - seg.r0 <= rt * kRowTile) {
          n += max(nt, 0);
          continue;
        }
        for (int j = 0; j < nt && ok; ++j, ++n) {
          const uint32_t st = n % kRing, buf = c & 1;
          // W first: with it the tile's stage is full and stays so until the arrival below
          ok = mbar_wait(w_full[2 * rt + buf], (c >> 1) & 1, kErr | 9, abort) &&
               mbar_wait(kv_full[st], (n / kRing) & 1, kErr | 7, abort);
          if (!ok) break;
          tc_fence_after();
          const uint64_t v = smem_desc_sw128(smem_u32(sm + L::oKV + st * 2 * L::kTileBytes + L::kTileBytes), kKeys * 128, 1024);
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i) mma_f16_ts(d, tmem + (2 * rt + buf) * kKeys + 8 * i, v + ((i * 2048) >> 4), idesc, j > 0 || i > 0);
          mma_commit(s_empty[2 * rt + buf]);
          mma_commit(kv_empty[st]);
          ++c;
        }
      }
    }
    // every MMA issued has completed before the tensor memory is freed
    mma_commit(drain[2 * rt + (scores ? 0 : 1)]);
    const long long start = clock64();
    while (!mbar_try_wait(drain[2 * rt + (scores ? 0 : 1)], 0) && clock64() - start < kWaitLimitCycles) {
    }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftWarps + kWideWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the line that CTA blockIdx.x began and did not finish (parts: slot 2 c + 1
// of that CTA, slot 2 c of the following ones; outputs as [D / 4][row] of four
// dims): a warp takes 16 dims of 32 rows, a row per lane, so that the parts are
// read whole and a lane writes 32 bytes.
template <int D>
__global__ void __launch_bounds__(32 * (D / 16)) paged_join_rows_kernel(const PagedAttendParams p, const PagedPartials ws,
                                                                        const bool bf16) {
  grid_dependents();
  grid_wait();
  const int c0 = blockIdx.x, dim = threadIdx.x >> 5, row = blockIdx.y * 32 + (threadIdx.x & 31);
  const PagedCut cut = ws.cut[c0];
  const int r = cut.row0 + row, R = p.b.H / p.c.G;
  if (cut.parts == 0 || r >= cut.nrows) return;
  float m = -INFINITY, M = -INFINITY, l = 0.f, acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll 2
  for (int k = 0; k < cut.parts; ++k) {
    const size_t slot = 2 * (size_t)(c0 + k) + (k == 0);
    const float4 h = ws.ml[slot * kRowsCta + row];
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = reinterpret_cast<const float4*>(ws.o)[(slot * (D / 4) + 4 * dim + i) * kRowsCta + row];
    const float mn = fmaxf(m, h.x), Mn = fmaxf(M, h.z);
    l = l * fast_exp2(m - finite_or_0(mn)) + h.y * fast_exp2(h.x - finite_or_0(mn));
    const float a = fast_exp2(M - finite_or_0(Mn)), b = fast_exp2(h.z - finite_or_0(Mn));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[4 * i] = acc[4 * i] * a + x[i].x * b;
      acc[4 * i + 1] = acc[4 * i + 1] * a + x[i].y * b;
      acc[4 * i + 2] = acc[4 * i + 2] * a + x[i].z * b;
      acc[4 * i + 3] = acc[4 * i + 3] * a + x[i].w * b;
    }
    m = mn;
    M = Mn;
  }
  const float inv = paged_normaliser(m, l, M);
  uint16_t* op = static_cast<uint16_t*>(p.out) + (int64_t)(cut.begin + r / R) * p.o_st +
                 (int64_t)(cut.g * R + r % R) * p.o_sh + 16 * dim;
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    uint32_t x[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      x[q] = bf16 ? pack2<__nv_bfloat16>(acc[i + 2 * q] * inv, acc[i + 2 * q + 1] * inv)
                  : pack2<__half>(acc[i + 2 * q] * inv, acc[i + 2 * q + 1] * inv);
    *reinterpret_cast<uint4*>(op + i) = make_uint4(x[0], x[1], x[2], x[3]);
  }
}

template <int KV, int D>
cudaError_t tc_launch(const PagedAttendParams& p, bool bf16, const PagedPartials& ws, int ctas, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may use its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !((allowed.load(std::memory_order_relaxed) >> dev) & 1)) {
    e = cudaFuncSetAttribute(paged_attend_tc_kernel<KV, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Lay<D>::bytes(kMaxBatch));
    if (e != cudaSuccess) return e;
    // the split of the registers holds for this launch allocation only: setmaxnreg.inc would wait for
    // registers that the block does not hold
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, paged_attend_tc_kernel<KV, D>);
    if (e != cudaSuccess) return e;
    if ((fa.numRegs + 7) / 8 * 8 != kRegs) return cudaErrorInvalidConfiguration;
    if (dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  e = launch_dependent(paged_attend_tc_kernel<KV, D>, dim3(ctas), kThreads, Lay<D>::bytes(p.b.B), st, p, ws, bf16);
  if (e != cudaSuccess) return e;
  return launch_dependent(paged_join_rows_kernel<D>, dim3(ctas, kRowsCta / 32), 32 * (D / 16), 0, st, p, ws, bf16);
}

}  // namespace

bool paged_attend_tc_takes(const PagedAttendParams& p) {
  const int R = p.b.H / p.c.G;
  if ((int64_t)p.b.max_tokens * R <= kTcRows || p.b.B > kMaxBatch) return false;
  const double lines = (double)p.b.T * R / kRowsCta + p.b.B;  // at most
  return lines * p.c.G * ((double)p.c.max_pages * p.c.page + p.b.max_tokens + kRowsCta + kLineCost) < 4e9;
}

size_t paged_attend_tc_workspace(const PagedAttendParams& p, int n_sm) {
  return paged_partials_bytes(n_sm, kRowsCta, p.c.D);
}

cudaError_t launch_paged_attend_tc(const PagedAttendParams& p, int dtype, int kv, void* ws, int n_sm,
                                   cudaStream_t st) {
  const PagedPartials s = paged_partials(ws, n_sm, kRowsCta);
  const bool bf16 = dtype == kBF16;
  if (p.c.D == 128)
    return kv == kKvInt8 ? tc_launch<kKvInt8, 128>(p, bf16, s, n_sm, st) : tc_launch<kKvE4m3, 128>(p, bf16, s, n_sm, st);
  if (p.c.D == 64)
    return kv == kKvInt8 ? tc_launch<kKvInt8, 64>(p, bf16, s, n_sm, st) : tc_launch<kKvE4m3, 64>(p, bf16, s, n_sm, st);
  return cudaErrorInvalidValue;
}

cudaError_t read_paged_device_error(unsigned int* code, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(code, sm100::g_device_error, sizeof(unsigned int));
  if (e != cudaSuccess || !reset) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(sm100::g_device_error, &zero, sizeof(unsigned int));
}

}  // namespace spatten
