// Joining the parts of a line of query rows that the work split of the paged
// attention kernels cut (paged_attend.cu, paged_attend_tc.cu).
#pragma once
#include "paged_dev.cuh"

namespace spatten {

// A line that a CTA begins and does not finish.
struct PagedCut {
  int parts;         // 0: none
  int row0, nrows;   // first row of the line among the sequence's, rows of the sequence
  int begin, g;      // first packed row of the sequence, KV head
  int pad[3];
};

struct PagedPartials {
  PagedCut* cut;  // [ctas]
  float4* ml;     // [2 ctas][rows] (m, l, M): slot 2 c: a line begun before CTA c; 2 c + 1: one begun in it
  float* o;       // [2 ctas][rows][D], by M
};

// The references of a row's exponentials follow its maxima where these have grown by
// more than kSlack: p = 2^(s - m) stays below 2^kSlack, and the f16 weights 2^(s +
// log2 v_scale - M), whose M is kRoom lower than its maximum, use f16's range up to
// 2^(kRoom + kSlack) = 2^15.
constexpr float kSlack = 8.f, kRoom = 7.f;
constexpr float kNoScale = -200.f;  // log2 of a scale of 0: below that of any float

SPATTEN_DEV float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }

// What takes an output by M to the result: 2^(M - m) / l, 0 for a row without a key.
SPATTEN_DEV float paged_normaliser(float m, float l, float M) {
  return l == 0.f ? 0.f : exp2f(fminf(finite_or_0(M) - finite_or_0(m), 127.f)) / l;
}

// Joins the line that CTA blockIdx.x began and did not finish: its parts are
// slot 2 c + 1 of that CTA and slot 2 c of the following ones. A warp per row
// and, where the line has fewer rows than the CTA has warps, per share of the
// parts; D / 32 dims per lane. Bound by the latency of its loads: the (m, l, M)
// of 64 parts (two per lane) and 8 outputs of the warp's share go out at once. It
// adds 5 us to a launch of its own, less under the programmatic dependence.
constexpr int kJoinWarps = 16;

template <int D, int ROWS>
__global__ void __launch_bounds__(32 * kJoinWarps, D == 128 ? 1 : 2)
paged_join_kernel(const PagedAttendParams p, const PagedPartials ws, const bool bf16) {
  constexpr int E = D / 32, FLY = 8, SPAN = 64;
  __shared__ float sh[kJoinWarps][D + 4];
  grid_dependents();
  grid_wait();
  const int c0 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PagedCut cut = ws.cut[c0];
  if (cut.parts == 0) return;
  const int R = p.b.H / p.c.G, rows = min(cut.nrows - cut.row0, ROWS);
  int share = kJoinWarps;  // warps per row
  while (share > 1 && rows * share > kJoinWarps) share >>= 1;
  const int row = warp / share, part0 = warp % share;
  const bool live = row < rows;
  auto at = [&](int i) { return (uint32_t)(2 * (c0 + i) + (i == 0)) * ROWS + row; };  // row of part i
  float m = -INFINITY, M = -INFINITY, l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int base = 0; live && base < cut.parts; base += SPAN) {
    const int end = min(base + SPAN, cut.parts);
    float4 h[2];  // of parts base + lane and base + 32 + lane
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = base + 32 * k + lane;
      h[k] = i < end ? ws.ml[at(i)] : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    }
    float f[2];
    for (int i0 = base + part0; i0 == base + part0 || i0 < end; i0 += FLY * share) {
      float x[FLY][E];
#pragma unroll
      for (int k = 0; k < FLY; ++k) {
        const int i = i0 + k * share;
        if (i < end) {
          const float* src = ws.o + (at(i) * D + lane * E);
          if constexpr (E == 4) {
            const float4 y = *reinterpret_cast<const float4*>(src);
            x[k][0] = y.x; x[k][1] = y.y; x[k][2] = y.z; x[k][3] = y.w;
          } else {
            const float2 y = *reinterpret_cast<const float2*>(src);
            x[k][0] = y.x; x[k][1] = y.y;
          }
        }
      }
      if (i0 == base + part0) {  // the span's weights, while the outputs are under way
        float mn = fmaxf(h[0].x, h[1].x), Mn = fmaxf(h[0].z, h[1].z);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
          mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
          Mn = fmaxf(Mn, __shfl_xor_sync(0xffffffffu, Mn, d));
        }
        mn = fmaxf(m, mn);
        Mn = fmaxf(M, Mn);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          f[k] = fast_exp2(h[k].z - finite_or_0(Mn));
          sum += h[k].y * fast_exp2(h[k].x - finite_or_0(mn));
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l = l * fast_exp2(m - finite_or_0(mn)) + sum;
        const float r = fast_exp2(M - finite_or_0(Mn));
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= r;
        m = mn;
        M = Mn;
      }
#pragma unroll
      for (int k = 0; k < FLY; ++k) {
        const int i = i0 + k * share;
        if (i >= end) break;  // warp-uniform
        const float w = __shfl_sync(0xffffffffu, i - base < 32 ? f[0] : f[1], (i - base) & 31);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += x[k][e] * w;
      }
    }
  }
  if (share > 1) {  // the shares of a row join in its first warp; each has the whole l
#pragma unroll
    for (int e = 0; e < E; ++e) sh[warp][lane * E + e] = acc[e];
    __syncthreads();
    if (part0 == 0)
      for (int w = 1; w < share; ++w) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += sh[warp + w][lane * E + e];
      }
  }
  if (live && part0 == 0) {
    const int r = cut.row0 + row;
    const float inv = paged_normaliser(m, l, M);
    uint16_t* op = static_cast<uint16_t*>(p.out) + (int64_t)(cut.begin + r / R) * p.o_st +
                   (int64_t)(cut.g * R + r % R) * p.o_sh + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2)
      *reinterpret_cast<uint32_t*>(op + e) =
          bf16 ? pack2<__nv_bfloat16>(acc[e] * inv, acc[e + 1] * inv) : pack2<__half>(acc[e] * inv, acc[e + 1] * inv);
  }
}

template <int D, int ROWS>
cudaError_t launch_paged_join(const PagedAttendParams& p, const PagedPartials& ws, int ctas, bool bf16,
                              cudaStream_t st) {
  static_assert(ROWS <= kJoinWarps, "a warp per row");
  return launch_dependent(paged_join_kernel<D, ROWS>, dim3(ctas), 32 * kJoinWarps, 0, st, p, ws, bf16);
}

inline size_t paged_align256(size_t x) { return (x + 255) & ~size_t(255); }

inline size_t paged_partials_bytes(size_t ctas, size_t rows, size_t D) {
  return paged_align256(ctas * sizeof(PagedCut)) + paged_align256(2 * ctas * rows * sizeof(float4)) +
         paged_align256(2 * ctas * rows * D * sizeof(float));
}

inline PagedPartials paged_partials(void* ws, size_t ctas, size_t rows) {
  uint8_t* w = static_cast<uint8_t*>(ws);
  PagedPartials s;
  s.cut = reinterpret_cast<PagedCut*>(w);
  w += paged_align256(ctas * sizeof(PagedCut));
  s.ml = reinterpret_cast<float4*>(w);
  w += paged_align256(2 * ctas * rows * sizeof(float4));
  s.o = reinterpret_cast<float*>(w);
  return s;
}

}  // namespace spatten
