// Device helpers shared by the kernels over the paged 8-bit KV cache.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"
#include "paged.h"

namespace spatten {

// Kernels over the cache follow one another many times a token, so each is
// launched as a dependent of the one before it in the stream (launch_dependent):
// its CTAs may start while the other's last ones run, and wait in grid_wait(),
// before any access to memory, until that grid is complete and its results are
// visible. grid_dependents() lets the next such launch start. Everything that a
// grid before may have written is read by plain loads: a read-only (nc) load may
// be moved ahead of the wait.
SPATTEN_DEV void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
SPATTEN_DEV void grid_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                             Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The packed rows [begin, begin + n) of sequence b, and the slot of the first:
// every value that comes from the device is brought into range here.
struct PagedSeq {
  int begin;  // first row of q / k / v / out
  int n;      // rows to process (at most max_tokens)
  int len;    // slots held, at most the page table's
  int old;    // slot of row `begin` (negative when seq_lens is below the row count)
};

SPATTEN_DEV PagedSeq paged_seq(const PagedBatch& p, const PagedCache& c, int b) {
  PagedSeq s;
  const int lo = *(p.cu + b), hi = *(p.cu + b + 1);
  const int len = min(max(*(p.lens + b), 0), 1 << 30);
  const int n = lo >= 0 && lo <= hi && hi <= p.T ? hi - lo : 0;  // rows out of order or range: none
  s.begin = n ? lo : 0;
  s.n = min(n, p.max_tokens);
  s.old = len - n;
  s.len = (int)min((int64_t)len, (int64_t)c.max_pages * c.page);
  return s;
}

// Whether a launch serves the sequence, given its query rows per KV head.
SPATTEN_DEV bool paged_serves(const PagedAttendParams& p, const PagedSeq& s, int R) {
  const int64_t rows = (int64_t)s.n * R;
  return rows > p.rows_over && rows <= p.rows_upto;
}

// Page of slots [pi * page, ...) of sequence b, or -1 where it has no memory.
SPATTEN_DEV int paged_page(const PagedCache& c, int b, int pi) {
  if (pi >= c.max_pages) return -1;
  const int pid = *(c.table + (int64_t)b * c.table_st + pi);
  return (pid >= 0 && pid < c.P) ? pid : -1;
}

// Bits j0 .. j0 + 31 of a row's words: whether the row sees the new tokens j0, ..;
// those before 0 are cached tokens, which every row sees.
SPATTEN_DEV uint32_t tree_bits(const uint32_t* w, int words, int j0) {
  const int i = j0 >> 5;
  auto word = [&](int k) { return k < 0 ? 0xFFFFFFFFu : k < words ? *(w + k) : 0u; };
  return __funnelshift_r(word(i), word(i + 1), j0 & 31);
}

// The statistics of a finished row, for the weights it gave: w = 2^(s - x) y.
SPATTEN_DEV float2 row_stat(float m, float l) {
  return make_float2(m == -INFINITY ? 0.f : m, l == 0.f ? 0.f : 1.f / l);
}

// Two e4m3 codes (low byte first) as f16x2; every e4m3 value is an f16.
SPATTEN_DEV uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("{ .reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t; }" : "=r"(r) : "r"(two));
  return r;
}

// Two floats as e4m3 codes, lo in the low byte: nearest even, saturated.
SPATTEN_DEV uint32_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
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

// Four codes (a 32-bit word, lowest byte first) as floats.
template <int KV>
SPATTEN_DEV void codes4_to_f32(uint32_t w, float (&f)[4]) {
  if constexpr (KV == kKvInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    const uint32_t a = e4m3x2_to_f16x2(w & 0xFFFFu), b = e4m3x2_to_f16x2(w >> 16);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
  }
}

// The same where the conversions' rate (a quarter of other instructions') is the bound, as
// in moves of cached tokens: an int8's byte x ^ 0x80 is the low one of the float 2^23 +
// 128 + code. (Reading back is bound by all instructions: 198 us with conversions, 218 so.)
template <int KV>
SPATTEN_DEV void codes4_to_f32_alu(uint32_t w, float (&f)[4]) {
  if constexpr (KV == kKvInt8) {
    const uint32_t x = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(x, 0x4B000000u, 0x7540 + i)) - 8388736.0f;
  } else {
    codes4_to_f32<KV>(w, f);
  }
}

// Eight earlier codes under a grown scale: round(code * ratio).
template <int KV>
SPATTEN_DEV uint2 rescale8(uint2 c, float ratio) {
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float f[4];
    codes4_to_f32_alu<KV>(j ? c.y : c.x, f);
    if constexpr (KV == kKvInt8) {
      uint32_t b[4];  // y + 1.5 2^23 holds the rounded y's low byte in its own
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(f[i], ratio), 12582912.0f));
      w[j] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      w[j] = f32x2_to_e4m3x2(f[0] * ratio, f[1] * ratio) | (f32x2_to_e4m3x2(f[2] * ratio, f[3] * ratio) << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}

// A query row as f16 for the product with the codes, times the power of two that
// takes its largest magnitude `top` to [2^14, 2^15): bf16 and fp16 values keep all
// their bits down to 2^-28 of that element, and some down to 2^-39 (powers of two
// that fp32 does not hold are left out: a row below 2^-112 stays smaller). A row
// that is not finite has no scores: its factor is NaN.
struct QueryScale {
  float up;      // the power
  float factor;  // what its scores are multiplied by, beside the key's scale
};

SPATTEN_DEV QueryScale query_scale(float top, float scale_log2) {
  const int e = top > 0.f ? 14 - max((int)(__float_as_uint(top) >> 23) - 127, -112) : 0;  // at most 126
  const float back = __uint_as_float((uint32_t)(127 - e) << 23);
  return {__uint_as_float((uint32_t)(127 + e) << 23), scale_log2 * back * (top <= 3.4e38f ? 1.f : NAN)};
}

}  // namespace spatten
