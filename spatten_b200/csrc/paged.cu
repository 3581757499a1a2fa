// Appending to and reading from the paged 8-bit KV cache.
//
// Append. A block (page, KV head) holds its tokens' codes and one scale:
//   int8:  S = max|x| / 127                     (IEEE division)
//   e4m3:  S = 2^ceil(log2(max|x| / 448))       (dividing by it is exact)
// A block's scale only grows: S' = max(S, that of the largest new magnitude);
// where it grew, the earlier codes become round(code * S / S'). Every step is
// a correctly rounded fp32 operation on its own (no contraction), and the
// sum of squares of the norm is taken in 64 bits, so that every order of it
// rounds to the same value: the codes do not depend on how lanes are arranged.
//
// One CTA per written block of K or V: the block's new rows stay in
// registers (8 dims per thread and row) between the maximum and the
// quantisation, so each input is read once and each code written once; the
// earlier codes are only touched where the scale grew. The query rows'
// norm and rotation ride in further CTAs of the same launch. A decode step is
// bound by the chain of dependent loads (lengths, page table, scale), a prompt
// by HBM.
#include "kernels.h"
#include "paged_dev.cuh"

namespace spatten {
namespace {

constexpr float kMaxFinite = 3.402823466e38f;

SPATTEN_DEV float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= kMaxFinite ? a : 0.f;  // infinities and NaN do not enter a scale
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

// Eight values over the block's scale, as codes.
template <int KV>
SPATTEN_DEV uint2 encode8(const float (&x)[8], float s) {
  uint32_t w[2] = {0u, 0u};
  if (s == 0.f) return make_uint2(0u, 0u);
  if constexpr (KV == kKvInt8) {
    const float rc = rcp_approx(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = min(max(quant_div(x[i], s, rc), -127), 127);  // NaN converts to 0
      w[i >> 2] |= ((uint32_t)c & 0xFFu) << (8 * (i & 3));
    }
  } else {
    const float inv = 1.0f / s;  // a power of two
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = x[i] == x[i] ? x[i] * inv : 0.f, b = x[i + 1] == x[i + 1] ? x[i + 1] * inv : 0.f;
      w[i >> 2] |= f32x2_to_e4m3x2(a, b) << (8 * (i & 3));
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
SPATTEN_DEV void load8(const T* p, float (&f)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(e[i]);
}

// Norm and rotation of one row spread over D / 8 lanes (lane li holds dims
// 8 li ..), all lanes of the warp taking part.
template <typename T, int D>
SPATTEN_DEV void norm_rotate(float (&x)[8], int li, const PagedAppendParams& p, const void* w, int pos) {
  constexpr int LPR = D / 8;
  if (w) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fma((double)x[i], (double)x[i], ss);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(__fadd_rn((float)(ss * (1.0 / D)), p.eps));
    float g[8];
    load8<T>(static_cast<const T*>(w) + li * 8, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], inv), g[i]);
  }
  if (p.cos) {
    const bool first = li < LPR / 2;
    const int64_t at = (int64_t)min(max(pos, 0), p.cs_rows - 1) * p.cs_st + (li % (LPR / 2)) * 8;
    float c[8], s[8];
    if (p.cs_f32) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.cos) + at) + j);
        const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.sin) + at) + j);
        c[4 * j] = a.x; c[4 * j + 1] = a.y; c[4 * j + 2] = a.z; c[4 * j + 3] = a.w;
        s[4 * j] = b.x; s[4 * j + 1] = b.y; s[4 * j + 2] = b.z; s[4 * j + 3] = b.w;
      }
    } else {
      load8<T>(static_cast<const T*>(p.cos) + at, c);
      load8<T>(static_cast<const T*>(p.sin) + at, s);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = __shfl_xor_sync(0xffffffffu, x[i], LPR / 2);  // the other half's value
      const float a = __fmul_rn(x[i], c[i]), b = __fmul_rn(y, s[i]);
      x[i] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
    }
  }
}

template <int D, int PAGE>
struct AppendShape {
  static constexpr int LPR = D / 8;                               // lanes per row
  static constexpr int NT = PAGE * D >= 8192 ? 256 : 128;         // threads
  static constexpr int RPP = NT / LPR;                            // rows per pass
  static constexpr int PASSES = PAGE / RPP;                       // at most 8: 64 values per thread
  static_assert(PASSES >= 1 && PASSES <= 8 && PAGE % RPP == 0, "a block's rows fit the registers");
};

// Grid (2 G + query CTAs, written blocks per sequence, B): unit x < G is K
// head x, x < 2 G V head x - G, the others share the chunk's query rows.
template <typename T, int KV, int D, int PAGE>
__global__ void __launch_bounds__(AppendShape<D, PAGE>::NT) paged_append_kernel(const PagedAppendParams p, int nqb) {
  using S = AppendShape<D, PAGE>;
  constexpr int LPR = S::LPR, RPP = S::RPP, PASSES = S::PASSES, NW = S::NT / 32;
  grid_dependents();
  grid_wait();
  const int b = blockIdx.z, chunk = blockIdx.y, G = p.c.G;
  const PagedSeq sq = paged_seq(p.b, p.c, b);
  if (sq.n == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, li = lane % LPR, rt = tid / LPR;

  if ((int)blockIdx.x >= 2 * G) {  // query rows of tokens [chunk * PAGE, ..): token-major, heads inside
    const int t0 = chunk * PAGE, rows = min(PAGE, sq.n - t0) * p.b.H;
    for (int r0 = ((int)blockIdx.x - 2 * G) * RPP; r0 < rows; r0 += nqb * RPP) {
      const int r = r0 + rt;
      const bool live = r < rows;
      const int i = t0 + (live ? r : 0) / p.b.H, h = (live ? r : 0) % p.b.H;
      const int64_t row = sq.begin + i;
      float x[8];
      load8<T>(static_cast<const T*>(p.q) + row * p.q_st + h * p.q_sh + li * 8, x);
      const int pos = p.positions ? __ldg(p.positions + row) : sq.old + i;
      norm_rotate<T, D>(x, li, p, p.wq, pos);
      if (live) {
        uint4 o;
        o.x = pack2<T>(x[0], x[1]); o.y = pack2<T>(x[2], x[3]);
        o.z = pack2<T>(x[4], x[5]); o.w = pack2<T>(x[6], x[7]);
        *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + row * p.qo_st + h * p.qo_sh + li * 8) = o;
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
  uint8_t* codes = (isk ? p.c.k : p.c.v) + blk * (PAGE * D) + li * 8;
  const float s_old = lo > 0 ? *sp : 0.f;
  const T* src = static_cast<const T*>(isk ? p.k : p.v) + g * (isk ? p.k_sh : p.v_sh) + li * 8;
  const int64_t st = isk ? p.k_st : p.v_st;

  float x[PASSES][8];
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < PASSES; ++j) {
    const int r = j * RPP + rt;
    const bool live = r >= lo && r < hi;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
    if (live) load8<T>(src + (int64_t)(sq.begin + first + r - sq.old) * st, x[j]);
  }
#pragma unroll
  for (int j = 0; j < PASSES; ++j) {
    const int r = j * RPP + rt;
    const bool live = r >= lo && r < hi;
    if (!__any_sync(0xffffffffu, live)) continue;
    if (isk) {
      const int64_t row = sq.begin + first + r - sq.old;
      const int pos = p.positions ? (live ? __ldg(p.positions + row) : 0) : first + r;
      norm_rotate<T, D>(x[j], li, p, p.wk, pos);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, live ? finite_abs(x[j][i]) : 0.f);
  }
  __shared__ float red[NW];
  amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));  // magnitudes order as integers
  if (lane == 0) red[tid >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) amax = fmaxf(amax, red[w]);
  const float s = fmaxf(s_old, scale_for<KV>(amax));
  if (s > s_old && lo > 0) {
    const float ratio = __fdiv_rn(s_old, s);
    for (int r = rt; r < lo; r += RPP) {
      uint2* c = reinterpret_cast<uint2*>(codes + r * D);
      *c = rescale8<KV>(*c, ratio);
    }
  }
#pragma unroll
  for (int j = 0; j < PASSES; ++j) {
    const int r = j * RPP + rt;
    if (r >= lo && r < hi) *reinterpret_cast<uint2*>(codes + r * D) = encode8<KV>(x[j], s);
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

// Read back: a thread per 16 codes of one (token, head) of K and of V, heads
// fastest, so that a warp writes consecutive 32-byte pieces and reads whole
// rows. Bound by HBM (1 byte in, 2 out).
template <typename T, int KV>
__global__ void __launch_bounds__(256) paged_read_kernel(const PagedReadParams p, int64_t total) {
  grid_dependents();
  grid_wait();
  const int lpr = p.c.D / 16, per_tok = p.c.G * lpr;
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= total) return;
  const int b = blockIdx.y;
  const int64_t j = t / per_tok;
  const int u = (int)(t % per_tok), g = u / lpr, d = (u % lpr) * 16;
  const int64_t slot = p.idx ? __ldg(p.idx + (int64_t)b * p.idx_st + j) : j;
  int pid = -1;
  if (slot >= 0 && slot < __ldg(p.lens + b) && slot < (int64_t)p.c.max_pages * p.c.page)
    pid = paged_page(p.c, b, (int)(slot / p.c.page));
  const int64_t blk = (int64_t)max(pid, 0) * p.c.G + g;
  const int64_t src = (blk * p.c.page + (pid < 0 ? 0 : slot % p.c.page)) * p.c.D + d;
  const int64_t dst = (((int64_t)b * p.N + j) * p.c.G + g) * p.c.D + d;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T* out = static_cast<T*>(which ? p.v_out : p.k_out);
    if (!out) continue;
    uint4 c = make_uint4(0u, 0u, 0u, 0u);
    float s = 0.f;
    if (pid >= 0) {
      c = *reinterpret_cast<const uint4*>((which ? p.c.v : p.c.k) + src);
      s = (which ? p.c.v_scale : p.c.k_scale)[blk];
    }
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
      codes4_to_f32<KV>(w[i], f);
      o[2 * i] = pack2<T>(f[0] * s, f[1] * s);
      o[2 * i + 1] = pack2<T>(f[2] * s, f[3] * s);
    }
    uint4* q = reinterpret_cast<uint4*>(out + dst);
    q[0] = make_uint4(o[0], o[1], o[2], o[3]);
    q[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

template <typename T, int KV>
cudaError_t read_launch(const PagedReadParams& p, cudaStream_t st) {
  const int64_t total = (int64_t)p.N * p.c.G * (p.c.D / 16);
  const dim3 grid((unsigned)((total + 255) / 256), p.B);
  return launch_dependent(paged_read_kernel<T, KV>, grid, 256, 0, st, p, total);
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
