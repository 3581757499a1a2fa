// Appending to and reading from the paged 8-bit KV cache.
//
// Append. A block (page, KV head) holds its tokens' codes and one scale:
//   int8:  S = max|x| / 127                     (IEEE division)
//   e4m3:  S = 2^ceil(log2(max|x| / 448))       (dividing by it is exact)
// A block's scale only grows: S' = max(S, that of the largest new magnitude);
// where it grew, the earlier codes become round(code * S / S'). Rotation and
// quantisation are correctly rounded fp32 operations one by one (no
// contraction); only the norm's sum of squares has an order of its own.
//
// One CTA per written block of K or V: the block's new rows stay in
// registers between the maximum and the quantisation, so each input is read
// once and each code written once; the earlier codes are only touched where the
// scale grew. A thread holds 4 dims of a row's first half and the 4 that rotate
// with them, so a rotation needs no exchange. The query rows' norm and rotation
// ride in further CTAs of the same launch. A decode step is bound by the chain
// of dependent loads (lengths, page table, scale): 2.6 us for one token, 5.2 us for
// 64 sequences. A prompt is bound by HBM and the issue slots (63 % of them used):
// 4 prompts of 8192 tokens (32 query, 8 KV heads, D = 128, bf16 to int8), 166 us =
// 4.46 TB/s, 0.68 of the measured copy rate.
#include "kernels.h"
#include "paged_dev.cuh"

namespace spatten {
namespace {

constexpr float kMaxFinite = 3.402823466e38f;

// The largest magnitude, NaN when one is.
SPATTEN_DEV float max_abs_nan(float a, float x, float y) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(x), "f"(y));
  return r;
}

// The scale that a block whose largest finite magnitude is `amax` needs.
template <int KV>
SPATTEN_DEV float scale_for(float amax) {
  if constexpr (KV == kKvInt8) {
    return div127_rn(amax);
  } else {
    if (amax == 0.f) return 0.f;
    // amax = m 2^e, m in [1, 2): 448 = 1.75 * 2^8, so k = e - 8, or e - 7 for m > 1.75
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127;  // -127 for subnormals, which the floor below covers
    const int k = max(e - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0), -126);
    return __uint_as_float((uint32_t)(k + 127) << 23);
  }
}

// Eight finite values over the block's scale (not 0), as codes; rc = 1 / s.
// int8: x rc (1 - 2^-20) and x rc (1 + 2^-20) enclose the rounded x / s, whose
// rounding is theirs where they agree; where one of the eight disagrees (near a
// tie, or with the infinity that a subnormal scale's reciprocal makes), they take
// the division. x rc + 1.5 2^23 holds the rounded integer's low byte in its own.
template <int KV>
SPATTEN_DEV uint2 encode8(const float2 (&x)[4], float s, float rc) {
  uint32_t w[2];
  if constexpr (KV == kKvInt8) {
    constexpr float kRound = 12582912.0f;
    const float below = rc * (1.f - 0x1p-20f), above = rc * (1.f + 0x1p-20f);
    const float2 r0 = make_float2(below, below), r1 = make_float2(above, above), up = make_float2(kRound, kRound);
    uint32_t b[8], differ = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __ffma2_rn(x[i], r0, up), t = __ffma2_rn(x[i], r1, up);
      b[2 * i] = __float_as_uint(f.x);
      b[2 * i + 1] = __float_as_uint(f.y);
      differ |= (b[2 * i] ^ __float_as_uint(t.x)) | (b[2 * i + 1] ^ __float_as_uint(t.y));
    }
    if (differ || !(above <= kMaxFinite)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[2 * i] = (uint32_t)__float2int_rn(__fdiv_rn(x[i].x, s));
        b[2 * i + 1] = (uint32_t)__float2int_rn(__fdiv_rn(x[i].y, s));
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      w[j] = __byte_perm(__byte_perm(b[4 * j], b[4 * j + 1], 0x0040), __byte_perm(b[4 * j + 2], b[4 * j + 3], 0x0040),
                         0x5410);
  } else {
    const float2 r2 = make_float2(rc, rc);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 a = __fmul2_rn(x[2 * j], r2), b = __fmul2_rn(x[2 * j + 1], r2);
      w[j] = f32x2_to_e4m3x2(a.x, a.y) | (f32x2_to_e4m3x2(b.x, b.y) << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}

// Eight earlier codes under a grown scale: round(code * ratio).
template <int KV>
SPATTEN_DEV uint2 rescale8(uint2 c, float ratio) {
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float f[4];
    codes4_to_f32<KV>(j ? c.y : c.x, f);
    if constexpr (KV == kKvInt8) {
      w[j] = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[j] |= ((uint32_t)__float2int_rn(f[i] * ratio) & 0xFFu) << (8 * i);
    } else {
      w[j] = f32x2_to_e4m3x2(f[0] * ratio, f[1] * ratio) | (f32x2_to_e4m3x2(f[2] * ratio, f[3] * ratio) << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}

template <typename T>
SPATTEN_DEV float2 unpack2(uint32_t u) {
  const T* e = reinterpret_cast<const T*>(&u);
  return make_float2(to_f32<T>(e[0]), to_f32<T>(e[1]));
}

// A lane's dims of a row: 4 li .. of its first half (f[0], f[1]) and of its second.
template <typename T, int D>
SPATTEN_DEV void load_halves(const T* row, int li, float2 (&f)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(row + 4 * li), b = *reinterpret_cast<const uint2*>(row + D / 2 + 4 * li);
  f[0] = unpack2<T>(a.x);
  f[1] = unpack2<T>(a.y);
  f[2] = unpack2<T>(b.x);
  f[3] = unpack2<T>(b.y);
}

// A lane's part of the rotation by a position: cos and sin of its pairs.
struct Turn {
  float2 c[2], s[2];
};

template <typename T>
SPATTEN_DEV void load_turn(Turn& r, const PagedAppendParams& p, int pos, int li) {
  const int64_t at = (int64_t)min(max(pos, 0), p.cs_rows - 1) * p.cs_st + 4 * li;
  if (p.cs_f32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p.cos) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p.sin) + at);
    r.c[0] = make_float2(a.x, a.y); r.c[1] = make_float2(a.z, a.w);
    r.s[0] = make_float2(b.x, b.y); r.s[1] = make_float2(b.z, b.w);
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const T*>(p.cos) + at);
    const uint2 b = *reinterpret_cast<const uint2*>(static_cast<const T*>(p.sin) + at);
    r.c[0] = unpack2<T>(a.x); r.c[1] = unpack2<T>(a.y);
    r.s[0] = unpack2<T>(b.x); r.s[1] = unpack2<T>(b.y);
  }
}

// Norm (g: the lane's weights) of one row spread over D / 8 lanes, all lanes of
// the warp taking part.
template <int D>
SPATTEN_DEV void norm_row(float2 (&x)[4], float eps, const float2 (&g)[4]) {
  float2 q = __fmul2_rn(x[0], x[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) q = __ffma2_rn(x[i], x[i], q);
  float ss = q.x + q.y;
#pragma unroll
  for (int o = D / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float inv = rsqrtf(__fadd_rn(ss * (1.0f / D), eps));
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __fmul2_rn(__fmul2_rn(x[i], make_float2(inv, inv)), g[i]);
}

SPATTEN_DEV void turn_row(float2 (&x)[4], const Turn& r) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = x[i], b = x[2 + i];
    x[i] = __fadd2_rn(__fmul2_rn(a, r.c[i]), __fmul2_rn(b, make_float2(-r.s[i].x, -r.s[i].y)));
    x[2 + i] = __fadd2_rn(__fmul2_rn(b, r.c[i]), __fmul2_rn(a, r.s[i]));
  }
}

template <int D, int PAGE>
struct AppendShape {
  static constexpr int LPR = D / 8;                               // lanes per row
  static constexpr int NT = PAGE * D >= 16384 ? 512 : PAGE * D >= 8192 ? 256 : 128;  // threads
  static constexpr int RPP = NT / LPR;                            // rows per pass
  static constexpr int PASSES = PAGE / RPP;                       // at most 4: 32 values per thread
  static_assert(PASSES >= 1 && PASSES <= 4 && PAGE % RPP == 0, "a block's rows fit the registers");
};

// Grid (2 G + query CTAs, written blocks per sequence, B): unit x < G is K
// head x, x < 2 G V head x - G, the others share the chunk's query rows.
template <typename T, int KV, int D, int PAGE, int HEADS>
__global__ void __launch_bounds__(AppendShape<D, PAGE>::NT, 1024 / AppendShape<D, PAGE>::NT)
paged_append_kernel(const PagedAppendParams p, int nqb) {
  using S = AppendShape<D, PAGE>;
  constexpr int LPR = S::LPR, RPP = S::RPP, PASSES = S::PASSES, NW = S::NT / 32;
  grid_dependents();
  grid_wait();
  const int b = blockIdx.z, chunk = blockIdx.y, G = p.c.G;
  const PagedSeq sq = paged_seq(p.b, p.c, b);
  if (sq.n == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, li = lane % LPR, rt = tid / LPR;

  if ((int)blockIdx.x >= 2 * G) {
    // query rows of tokens [chunk * PAGE, ..): a row of lanes takes HEADS heads of a token, which share
    // its rotation and are in flight together
    const int t0 = chunk * PAGE, H = p.b.H, groups = (H + HEADS - 1) / HEADS;
    const int items = min(PAGE, sq.n - t0) * groups;
    float2 w[4];
    if (p.wq) load_halves<T, D>(static_cast<const T*>(p.wq), li, w);
    for (int i0 = ((int)blockIdx.x - 2 * G) * RPP; i0 < items; i0 += nqb * RPP) {
      const bool live = i0 + rt < items;
      const int item = live ? i0 + rt : items - 1, tok = t0 + item / groups, h0 = item % groups * HEADS;
      const int64_t row = sq.begin + tok;
      const T* src = static_cast<const T*>(p.q) + row * p.q_st + h0 * p.q_sh;
      T* dst = static_cast<T*>(p.q_out) + row * p.qo_st + h0 * p.qo_sh + 4 * li;
      Turn turn;
      if (p.cos) load_turn<T>(turn, p, p.positions ? p.positions[row] : sq.old + tok, li);
      float2 x[HEADS][4];
#pragma unroll
      for (int h = 0; h < HEADS; ++h) load_halves<T, D>(src + min(h, H - 1 - h0) * p.q_sh, li, x[h]);
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        if (p.wq) norm_row<D>(x[h], p.eps, w);
        if (p.cos) turn_row(x[h], turn);
        if (live && h0 + h < H) {
          T* o = dst + h * p.qo_sh;
          *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(x[h][0].x, x[h][0].y), pack2<T>(x[h][1].x, x[h][1].y));
          *reinterpret_cast<uint2*>(o + D / 2) =
              make_uint2(pack2<T>(x[h][2].x, x[h][2].y), pack2<T>(x[h][3].x, x[h][3].y));
        }
      }
    }
    return;
  }

  const bool isk = (int)blockIdx.x < G;
  const int g = isk ? blockIdx.x : blockIdx.x - G;
  const int pi = max(sq.old, 0) / PAGE + chunk, first = pi * PAGE;
  if (pi >= p.c.max_pages) return;
  // new rows [lo, hi) of the block; earlier ones [0, lo)
  const int lo = max(sq.old - first, 0), hi = min(min(sq.old + sq.n, sq.len) - first, PAGE);
  if (hi <= lo) return;
  const int pid = paged_page(p.c, b, pi);
  if (pid < 0) return;
  const int64_t blk = (int64_t)pid * G + g;
  float* sp = (isk ? p.c.k_scale : p.c.v_scale) + blk;
  uint8_t* codes = (isk ? p.c.k : p.c.v) + blk * (PAGE * D);
  const float s_old = lo > 0 ? *sp : 0.f;
  const int64_t st = isk ? p.k_st : p.v_st;
  const int64_t row0 = sq.begin + first - sq.old;  // packed row of the block's row 0
  const T* src = static_cast<const T*>(isk ? p.k : p.v) + row0 * st + g * (isk ? p.k_sh : p.v_sh);

  float2 x[PASSES][4];  // rows that are not new: zeros
#pragma unroll
  for (int j = 0; j < PASSES; ++j) {
    const int r = j * RPP + rt;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[j][i] = make_float2(0.f, 0.f);
    if (r >= lo && r < hi) load_halves<T, D>(src + r * st, li, x[j]);
  }
  float amax = 0.f;
  if (isk && (p.wk || p.cos)) {
    float2 w[4];
    if (p.wk) load_halves<T, D>(static_cast<const T*>(p.wk), li, w);
    // a pass ahead where there are several: a row's rotation is a load of its own
    Turn ahead;
    auto used = [&](int j) { return j < PASSES && hi > j * RPP && lo < (j + 1) * RPP; };
    auto fetch = [&](int j) {
      const int r = j * RPP + rt;
      load_turn<T>(ahead, p, p.positions ? (r >= lo && r < hi ? p.positions[row0 + r] : 0) : first + r, li);
    };
    constexpr int EARLY = HEADS > 1 ? 1 : 0;
    if (EARLY && p.cos && used(0)) fetch(0);
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      Turn turn = ahead;
      if (p.cos && used(j + EARLY)) fetch(j + EARLY);
      if (!EARLY) turn = ahead;
      if (used(j)) {
        if (p.wk) norm_row<D>(x[j], p.eps, w);
        if (p.cos) turn_row(x[j], turn);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < PASSES; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = max_abs_nan(amax, x[j][i].x, x[j][i].y);
  __shared__ float red[NW];
  // magnitudes order as integers, NaN above infinity above the rest
  auto reduce = [&]() {
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
    if (lane == 0) red[tid >> 5] = __uint_as_float(top);
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) all = max(all, __float_as_uint(red[w]));
    amax = __uint_as_float(all);
  };
  reduce();
  bool odd = !(amax <= kMaxFinite);
  if (odd) {  // they do not enter the scale: the largest of the rest
    amax = 0.f;
#pragma unroll
    for (int j = 0; j < PASSES; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = fabsf(i & 1 ? x[j][i >> 1].y : x[j][i >> 1].x);
        if (a <= kMaxFinite) amax = fmaxf(amax, a);
      }
    __syncthreads();
    reduce();
  }
  const float s = fmaxf(s_old, scale_for<KV>(amax));
  if (odd) {  // a NaN is stored as 0, an infinity as the largest code of its sign
    const float top = s * (KV == kKvInt8 ? 127.f : 448.f);
#pragma unroll
    for (int j = 0; j < PASSES; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float& y = i & 1 ? x[j][i >> 1].y : x[j][i >> 1].x;
        if (!(fabsf(y) <= kMaxFinite)) y = y == y ? copysignf(top, y) : 0.f;
      }
  }
  if (s > s_old && lo > 0) {
    const float ratio = __fdiv_rn(s_old, s);
    for (int r = rt; r < lo; r += RPP) {
      uint2* c = reinterpret_cast<uint2*>(codes + r * D + 8 * li);
      *c = rescale8<KV>(*c, ratio);
    }
  }
  const float rc = KV == kKvInt8 ? rcp_approx(s) : 1.0f / s;  // e4m3: a power of two
#pragma unroll
  for (int j = 0; j < PASSES; ++j) {
    const int r = j * RPP + rt;
    if (r >= lo && r < hi) {
      const uint2 c = s > 0.f ? encode8<KV>(x[j], s, rc) : make_uint2(0u, 0u);
      *reinterpret_cast<uint32_t*>(codes + r * D + 4 * li) = c.x;
      *reinterpret_cast<uint32_t*>(codes + r * D + D / 2 + 4 * li) = c.y;
    }
  }
  if (tid == 0) *sp = s;
}

template <typename T, int KV, int D, int PAGE, int HEADS>
cudaError_t append_heads(const PagedAppendParams& p, int passes, cudaStream_t st) {
  using S = AppendShape<D, PAGE>;
  const int mt = p.b.max_tokens;
  const int chunks = (int)(((int64_t)mt + PAGE - 2) / PAGE + 1);  // mt tokens touch at most this many blocks
  int nqb = 0;
  if (p.q) {
    const int64_t items = (int64_t)(mt < PAGE ? mt : PAGE) * ((p.b.H + HEADS - 1) / HEADS);
    nqb = (int)((items + S::RPP * passes - 1) / (S::RPP * passes));
  }
  return launch_dependent(paged_append_kernel<T, KV, D, PAGE, HEADS>, dim3(2 * p.c.G + nqb, chunks, p.b.B), S::NT, 0,
                          st, p, nqb);
}

// A few tokens: a head per row of lanes, one pass per CTA (latency). Prompts:
// four heads share a token's rotation (two at a time: 168 -> 182 us at 4 prompts
// of 8192 tokens), two passes the set-up (one: 173 us). The first form against the
// second (32/8 heads x 128): one sequence of 1, 15, 32 and 64 tokens 2.6, 2.6, 3.3 and
// 4.2 us against 2.7, 3.7, 3.8 and 4.5; 8 sequences of 15, 32 and 64 3.7, 5.1 and 7.8
// against 4.7, 5.8 and 6.7; 64 of 1, 4, 8, 15 and 32 5.4, 8.1, 9.9, 15.3 and 23.4
// against 5.8, 8.1, 9.1, 13.0 and 16.9. The border lies between where 64 sequences
// and where one would have it.
template <typename T, int KV, int D, int PAGE>
cudaError_t append_launch(const PagedAppendParams& p, cudaStream_t st) {
  return p.b.max_tokens < 16 ? append_heads<T, KV, D, PAGE, 1>(p, 1, st) : append_heads<T, KV, D, PAGE, 4>(p, 2, st);
}

template <typename T, int KV, int D>
cudaError_t append_page(const PagedAppendParams& p, cudaStream_t st) {
  switch (p.c.page) {
    case 16: return append_launch<T, KV, D, 16>(p, st);
    case 32: return append_launch<T, KV, D, 32>(p, st);
    case 64: return append_launch<T, KV, D, 64>(p, st);
    case 128: return append_launch<T, KV, D, 128>(p, st);
    default: return cudaErrorInvalidValue;
  }
}

template <typename T, int KV>
cudaError_t append_dim(const PagedAppendParams& p, cudaStream_t st) {
  if (p.c.D == 128) return append_page<T, KV, 128>(p, st);
  if (p.c.D == 64) return append_page<T, KV, 64>(p, st);
  return cudaErrorInvalidValue;
}

// Read back. A CTA takes a run of tokens of one sequence; a thread takes 8 codes
// of one (token, head) of K and of V at a time, heads fastest, so that a warp
// reads whole rows and writes consecutive 16-byte pieces, and has four of them in
// flight (index, page and codes each wait for the one before). Bound by HBM
// (1 byte in, 2 out): 2048 of 8192 tokens of 64 sequences, 154 us = 5.23 TB/s, 0.80 of
// the measured copy rate.
constexpr int kReadThreads = 256, kReadFly = 4;

template <typename T, int KV>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const PagedReadParams p, int tokens) {
  grid_dependents();
  grid_wait();
  const int lpr = p.c.D / 8, per = p.c.G * lpr, b = blockIdx.y;
  const int64_t j0 = (int64_t)blockIdx.x * tokens;
  const int items = (int)min((int64_t)tokens, p.N - j0) * per;
  const int64_t len = min((int64_t)*(p.lens + b), (int64_t)p.c.max_pages * p.c.page);
  const int page_log = __ffs(p.c.page) - 1;
  for (int i0 = threadIdx.x; i0 < items; i0 += kReadThreads * kReadFly) {
    int64_t slot[kReadFly];
    int u[kReadFly], pid[kReadFly];
#pragma unroll
    for (int f = 0; f < kReadFly; ++f) {
      const int i = min(i0 + f * kReadThreads, items - 1);
      const int64_t j = j0 + i / per;
      u[f] = i % per;
      slot[f] = p.idx ? *(p.idx + (int64_t)b * p.idx_st + j) : j;
    }
#pragma unroll
    for (int f = 0; f < kReadFly; ++f)
      pid[f] = slot[f] >= 0 && slot[f] < len ? paged_page(p.c, b, (int)(slot[f] >> page_log)) : -1;
    uint2 c[kReadFly][2];
    float s[kReadFly][2];
#pragma unroll
    for (int f = 0; f < kReadFly; ++f) {
      const int64_t blk = (int64_t)max(pid[f], 0) * p.c.G + u[f] / lpr;
      const int64_t src = (blk * p.c.page + (slot[f] & (p.c.page - 1))) * p.c.D + u[f] % lpr * 8;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        c[f][w] = make_uint2(0u, 0u);
        s[f][w] = 0.f;
        if (pid[f] >= 0 && (w ? p.v_out : p.k_out)) {
          c[f][w] = *(reinterpret_cast<const uint2*>((w ? p.c.v : p.c.k) + src));
          s[f][w] = *((w ? p.c.v_scale : p.c.k_scale) + blk);
        }
      }
    }
#pragma unroll
    for (int f = 0; f < kReadFly; ++f) {
      const int i = i0 + f * kReadThreads;
      if (i >= items) break;
      const int64_t dst = (((int64_t)b * p.N + j0) * per + i) * 8;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        T* out = static_cast<T*>(w ? p.v_out : p.k_out);
        if (!out) continue;
        float x[4], y[4];
        codes4_to_f32<KV>(c[f][w].x, x);
        codes4_to_f32<KV>(c[f][w].y, y);
        const float m = s[f][w];
        *reinterpret_cast<uint4*>(out + dst) =
            make_uint4(pack2<T>(x[0] * m, x[1] * m), pack2<T>(x[2] * m, x[3] * m), pack2<T>(y[0] * m, y[1] * m),
                       pack2<T>(y[2] * m, y[3] * m));
      }
    }
  }
}

template <typename T, int KV>
cudaError_t read_launch(const PagedReadParams& p, cudaStream_t st) {
  const int per = p.c.G * (p.c.D / 8), run = kReadThreads * kReadFly;
  const int tokens = per < run ? run / per : 1;
  const dim3 grid((unsigned)((p.N + (int64_t)tokens - 1) / tokens), p.B);
  return launch_dependent(paged_read_kernel<T, KV>, grid, kReadThreads, 0, st, p, tokens);
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& p, int dtype, int kv, cudaStream_t st) {
  if (dtype == kF16) return kv == kKvInt8 ? append_dim<__half, kKvInt8>(p, st) : append_dim<__half, kKvE4m3>(p, st);
  if (dtype == kBF16)
    return kv == kKvInt8 ? append_dim<__nv_bfloat16, kKvInt8>(p, st) : append_dim<__nv_bfloat16, kKvE4m3>(p, st);
  return cudaErrorInvalidValue;
}

cudaError_t launch_paged_read(const PagedReadParams& p, int dtype, int kv, cudaStream_t st) {
  if (dtype == kF16) return kv == kKvInt8 ? read_launch<__half, kKvInt8>(p, st) : read_launch<__half, kKvE4m3>(p, st);
  if (dtype == kBF16)
    return kv == kKvInt8 ? read_launch<__nv_bfloat16, kKvInt8>(p, st) : read_launch<__nv_bfloat16, kKvE4m3>(p, st);
  return cudaErrorInvalidValue;
}

}  // namespace spatten
