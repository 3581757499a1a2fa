// Attention over the paged 8-bit KV cache (spatten_paged_attend).
//
// Online softmax over the slots that a query sees: a warp per (query row,
// head), D / 32 dims per lane, one key at a time:
//   s = sm_scale * k_scale * (q . k_codes),  m' = max(m, s),
//   l = l 2^(m - m') + 2^(s - m'),  o = o 2^(m - m') + 2^(s - m') v_scale v_codes
// in fp32 and the log2 domain; o / l, or 0 where no slot is seen.
#include "kernels.h"
#include "paged_dev.cuh"

namespace spatten {
namespace {

template <typename T, int KV, int D>
__global__ void __launch_bounds__(128) paged_attend_kernel(const PagedAttendParams p) {
  constexpr int E = D / 32;
  const int b = blockIdx.z, i = blockIdx.x, lane = threadIdx.x & 31;
  const int h = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const PagedSeq sq = paged_seq(p.b, p.c, b);
  if (i >= sq.n || h >= p.b.H) return;
  const int g = h / (p.b.H / p.c.G), page = p.c.page;
  const int64_t row = sq.begin + i;
  const T* qp = static_cast<const T*>(p.q) + row * p.q_st + h * p.q_sh + lane * E;
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = to_f32<T>(qp[e]) * p.scale_log2;
    o[e] = 0.f;
  }
  const int limit = min(sq.old + i + 1, sq.len);
  for (int n = 0; n < limit; ++n) {
    const int pid = paged_page(p.c, b, n / page);
    if (pid < 0) continue;
    const int64_t blk = (int64_t)pid * p.c.G + g, at = (blk * page + n % page) * D + lane * E;
    uint32_t kw = 0, vw = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      kw |= (uint32_t)p.c.k[at + e] << (8 * e);
      vw |= (uint32_t)p.c.v[at + e] << (8 * e);
    }
    float kf[4], vf[4], s = 0.f;
    codes4_to_f32<KV>(kw, kf);
    codes4_to_f32<KV>(vw, vf);
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * kf[e];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.c.k_scale[blk];
    const float mn = fmaxf(m, s), a = exp2f(m - mn), w = exp2f(s - mn), vs = p.c.v_scale[blk] * w;
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + vs * vf[e];
    m = mn;
  }
  T* op = static_cast<T*>(p.out) + row * p.o_st + h * p.o_sh + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = from_f32<T>(l > 0.f ? o[e] / l : (l == l ? 0.f : l));
}

template <typename T, int KV>
cudaError_t attend_dim(const PagedAttendParams& p, cudaStream_t st) {
  const dim3 grid(p.b.max_tokens, (p.b.H + 3) / 4, p.b.B);
  if (p.c.D == 128) paged_attend_kernel<T, KV, 128><<<grid, 128, 0, st>>>(p);
  else if (p.c.D == 64) paged_attend_kernel<T, KV, 64><<<grid, 128, 0, st>>>(p);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

}  // namespace

size_t paged_attend_workspace(const PagedAttendParams&, int) { return 0; }

cudaError_t launch_paged_attend(const PagedAttendParams& p, int dtype, int kv, void*, int, cudaStream_t st) {
  if (dtype == kF16) return kv == kKvInt8 ? attend_dim<__half, kKvInt8>(p, st) : attend_dim<__half, kKvE4m3>(p, st);
  if (dtype == kBF16)
    return kv == kKvInt8 ? attend_dim<__nv_bfloat16, kKvInt8>(p, st) : attend_dim<__nv_bfloat16, kKvE4m3>(p, st);
  return cudaErrorInvalidValue;
}

}  // namespace spatten
