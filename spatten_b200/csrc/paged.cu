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
// of dependent loads (lengths, page table, scale), a prompt by HBM and the
// instructions per element.
#include "kernels.h"
#include "paged_dev.cuh"

namespace spatten {
namespace {

constexpr float kMaxFinite = 3.402823466e38f;

// The larger magnitude, NaN when either is.
SPATTEN_DEV float max_abs_nan(float a, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(x)));
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
template <int KV>
SPATTEN_DEV uint2 encode8(const float (&x)[8], float s, float rc) {
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (KV == kKvInt8) {
      int c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = quant_div_fadd(x[4 * j + i], s, rc);
      const uint32_t lo = __byte_perm(c[0], c[1], 0x0040), hi = __byte_perm(c[2], c[3], 0x0040);
      w[j] = __byte_perm(lo, hi, 0x5410);
    } else {
      w[j] = f32x2_to_e4m3x2(x[4 * j] * rc, x[4 * j + 1] * rc) |
             (f32x2_to_e4m3x2(x[4 * j + 2] * rc, x[4 * j + 3] * rc) << 16);
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
SPATTEN_DEV void unpack4(uint2 u, float* f) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = to_f32<T>(e[i]);
}

// A lane's dims of a row: 4 li .. of its first half (f[0 .. 3]) and of its second.
template <typename T, int D>
SPATTEN_DEV void load_halves(const T* row, int li, float (&f)[8]) {
  unpack4<T>(*(reinterpret_cast<const uint2*>(row + 4 * li)), f);
  unpack4<T>(*(reinterpret_cast<const uint2*>(row + D / 2 + 4 * li)), f + 4);
}

// Norm and rotation of one row spread over D / 8 lanes, all lanes of the warp
// taking part; g: the lane's norm weights.
template <typename T, int D>
SPATTEN_DEV void norm_rotate(float (&x)[8], int li, const PagedAppendParams& p, const float* g, int pos) {
  if (g) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(__fadd_rn(ss * (1.0f / D), p.eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], inv), g[i]);
  }
  if (p.cos) {
    const int64_t at = (int64_t)min(max(pos, 0), p.cs_rows - 1) * p.cs_st + 4 * li;
    float c[4], s[4];
    if (p.cs_f32) {
      const float4 a = *(reinterpret_cast<const float4*>(static_cast<const float*>(p.cos) + at));
      const float4 b = *(reinterpret_cast<const float4*>(static_cast<const float*>(p.sin) + at));
      c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w;
      s[0] = b.x; s[1] = b.y; s[2] = b.z; s[3] = b.w;
    } else {
      unpack4<T>(*(reinterpret_cast<const uint2*>(static_cast<const T*>(p.cos) + at)), c);
      unpack4<T>(*(reinterpret_cast<const uint2*>(static_cast<const T*>(p.sin) + at)), s);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[i], b = x[4 + i];
      x[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
      x[4 + i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
    }
  }
}

template <int D, int PAGE>
struct AppendShape {
  static constexpr int LPR = D / 8;                               // lanes per row
  static constexpr int NT = PAGE * D >= 16384 ? 512 : PAGE * D >= 8192 ? 256 : 128;  // threads
  static constexpr int RPP = NT / LPR;                            // rows per pass
  static constexpr int PASSES = PAGE / RPP;                       // at most 4: 32 values per thread
  static constexpr int QROWS = 2;                                 // query rows of a thread in flight
  static_assert(PASSES >= 1 && PASSES <= 4 && PAGE % RPP == 0, "a block's rows fit the registers");
};

// Grid (2 G + query CTAs, written blocks per sequence, B): unit x < G is K
// head x, x < 2 G V head x - G, the others share the chunk's query rows.
template <typename T, int KV, int D, int PAGE>
__global__ void __launch_bounds__(AppendShape<D, PAGE>::NT, 1024 / AppendShape<D, PAGE>::NT)
paged_append_kernel(const PagedAppendParams p, int nqb) {
  using S = AppendShape<D, PAGE>;
  constexpr int LPR = S::LPR, RPP = S::RPP, PASSES = S::PASSES, NW = S::NT / 32, QR = S::QROWS;
  grid_dependents();
  grid_wait();
  const int b = blockIdx.z, chunk = blockIdx.y, G = p.c.G;
  const PagedSeq sq = paged_seq(p.b, p.c, b);
  if (sq.n == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, li = lane % LPR, rt = tid / LPR;

  if ((int)blockIdx.x >= 2 * G) {  // query rows of tokens [chunk * PAGE, ..): token-major, heads inside
    const int t0 = chunk * PAGE, H = p.b.H, rows = min(PAGE, sq.n - t0) * H;
    float w[8];
    if (p.wq) load_halves<T, D>(static_cast<const T*>(p.wq), li, w);
    for (int r0 = ((int)blockIdx.x - 2 * G) * RPP; r0 < rows; r0 += nqb * RPP * QR) {
      float x[QR][8];
      int tok[QR], h[QR];
#pragma unroll
      for (int j = 0; j < QR; ++j) {
        const int r = min(r0 + j * nqb * RPP + rt, rows - 1);
        tok[j] = t0 + r / H;
        h[j] = r % H;
        load_halves<T, D>(static_cast<const T*>(p.q) + (sq.begin + tok[j]) * p.q_st + h[j] * p.q_sh, li, x[j]);
      }
#pragma unroll
      for (int j = 0; j < QR; ++j) {
        if (r0 + j * nqb * RPP >= rows) break;  // uniform
        const int64_t row = sq.begin + tok[j];
        norm_rotate<T, D>(x[j], li, p, p.wq ? w : nullptr, p.positions ? *(p.positions + row) : sq.old + tok[j]);
        if (r0 + j * nqb * RPP + rt < rows) {
          T* o = static_cast<T*>(p.q_out) + row * p.qo_st + h[j] * p.qo_sh + 4 * li;
          *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(x[j][0], x[j][1]), pack2<T>(x[j][2], x[j][3]));
          *reinterpret_cast<uint2*>(o + D / 2) = make_uint2(pack2<T>(x[j][4], x[j][5]), pack2<T>(x[j][6], x[j][7]));
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

  float x[PASSES][8];  // rows that are not new: zeros
#pragma unroll
  for (int j = 0; j < PASSES; ++j) {
    const int r = j * RPP + rt;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
    if (r >= lo && r < hi) load_halves<T, D>(src + r * st, li, x[j]);
  }
  float amax = 0.f;
  if (isk && (p.wk || p.cos)) {
    float w[8];
    if (p.wk) load_halves<T, D>(static_cast<const T*>(p.wk), li, w);
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      const int r = j * RPP + rt;
      const bool live = r >= lo && r < hi;
      if (__any_sync(0xffffffffu, live))
        norm_rotate<T, D>(x[j], li, p, p.wk ? w : nullptr,
                          p.positions ? (live ? *(p.positions + row0 + r) : 0) : first + r);
    }
  }
#pragma unroll
  for (int j = 0; j < PASSES; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_abs_nan(amax, x[j][i]);
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
        const float a = fabsf(x[j][i]);
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
      for (int i = 0; i < 8; ++i)
        if (!(fabsf(x[j][i]) <= kMaxFinite)) x[j][i] = x[j][i] == x[j][i] ? copysignf(top, x[j][i]) : 0.f;
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

template <typename T, int KV, int D, int PAGE>
cudaError_t append_launch(const PagedAppendParams& p, cudaStream_t st) {
  using S = AppendShape<D, PAGE>;
  const int mt = p.b.max_tokens;
  const int chunks = (int)(((int64_t)mt + PAGE - 2) / PAGE + 1);  // mt tokens touch at most this many blocks
  int nqb = 0;
  if (p.q) {
    // a few tokens: one pass per CTA (latency); prompts: eight, to amortise the set-up
    const int64_t rows = (int64_t)(mt < PAGE ? mt : PAGE) * p.b.H;
    const int per = S::RPP * (mt < 16 ? 1 : 8);
    nqb = (int)((rows + per - 1) / per);
  }
  return launch_dependent(paged_append_kernel<T, KV, D, PAGE>, dim3(2 * p.c.G + nqb, chunks, p.b.B), S::NT, 0, st, p,
                          nqb);
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
// (1 byte in, 2 out).
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
