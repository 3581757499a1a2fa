// The weights that the new tokens give the cached ones (spatten_paged_attend_ext
// with weights): after the attention, whose statistics (m, 1 / l) of each row are
// read,
//   weight[slot] = (slot is an earlier token's ? weight[slot] : 0) + sum over rows
//                  of 2^(q . k sm_scale log2(e) - m) / l
// for every slot that a row of the call may see; the new tokens' slots take their
// positions.
//
// A thread holds the key of a slot and walks the rows, which it reads from shared
// memory.
#include "kernels.h"
#include "paged_dev.cuh"

namespace spatten {
namespace {

constexpr int kSlots = 128, kRows = 16;

template <typename T, int KV, int D>
__global__ void __launch_bounds__(kSlots) paged_weigh_kernel(const PagedWeighParams p) {
  __shared__ __align__(16) float q[kRows][D];
  __shared__ float2 stat[kRows];
  grid_dependents();
  grid_wait();
  const PagedAttendParams& a = p.a;
  const int b = blockIdx.z, g = blockIdx.y, G = a.c.G, R = a.b.H / G, page = a.c.page, tid = threadIdx.x;
  const PagedSeq sq = paged_seq(a.b, a.c, b);
  const int first = blockIdx.x * kSlots, slot = first + tid, lim = min(sq.old + sq.n, sq.len);
  if (sq.n == 0 || first >= lim || sq.n * R <= p.rows_over) return;
  const int pid = slot < lim ? paged_page(a.c, b, slot / page) : -1;
  const int64_t row = ((int64_t)max(pid, 0) * G + g) * page + slot % page;
  float k[D], ks = 0.f;
#pragma unroll
  for (int d = 0; d < D; ++d) k[d] = 0.f;
  if (pid >= 0) {
    const uint4* src = reinterpret_cast<const uint4*>(a.c.k + row * D);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint4 w = src[i];
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[4];
        codes4_to_f32<KV>(x[j], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) k[16 * i + 4 * j + e] = f[e];
      }
    }
    ks = a.c.k_scale[(int64_t)pid * G + g] * a.scale_log2;
  }
  float sum = 0.f;
  const int nrows = sq.n * R;
  for (int r0 = 0; r0 < nrows; r0 += kRows) {
    __syncthreads();
    for (int i = tid; i < kRows * D; i += kSlots) {
      const int r = r0 + i / D;
      if (r < nrows)
        q[i / D][i % D] = to_f32<T>(static_cast<const T*>(a.q)[(int64_t)(sq.begin + r / R) * a.q_st +
                                                                (int64_t)(g * R + r % R) * a.q_sh + i % D]);
    }
    if (tid < kRows && r0 + tid < nrows)
      stat[tid] = a.stat[(int64_t)(sq.begin + (r0 + tid) / R) * a.b.H + g * R + (r0 + tid) % R];
    __syncthreads();
    for (int j = 0; j < min(kRows, nrows - r0); ++j) {
      const int i = (r0 + j) / R;
      const bool sees = a.tree ? slot < sq.old || (tree_bits(a.tree + (sq.begin + i) * a.tree_st, a.words, slot - sq.old) & 1u)
                               : slot < sq.old + i + 1;
      float s = 0.f;
#pragma unroll
      for (int d = 0; d < D; d += 4) {
        const float4 x = *reinterpret_cast<const float4*>(&q[j][d]);
        s = fmaf(x.x, k[d], s);
        s = fmaf(x.y, k[d + 1], s);
        s = fmaf(x.z, k[d + 2], s);
        s = fmaf(x.w, k[d + 3], s);
      }
      if (sees) sum += exp2f(s * ks - stat[j].x) * stat[j].y;
    }
  }
  if (pid < 0) return;
  p.weight[row] = (slot < sq.old ? p.weight[row] : 0.f) + sum;
  if (slot >= sq.old)
    p.position[row] = p.positions ? p.positions[sq.begin + slot - sq.old] : slot;
}

// Sequences of few rows, whose scores the attention kept: a thread per slot, all heads.
constexpr int kScoreThreads = 256;

template <int ROWS>
__global__ void __launch_bounds__(kScoreThreads) paged_weigh_scores_kernel(const PagedWeighParams p) {
  grid_dependents();
  grid_wait();
  const PagedAttendParams& a = p.a;
  const int b = blockIdx.y, G = a.c.G, R = a.b.H / G, page = a.c.page;
  const PagedSeq sq = paged_seq(a.b, a.c, b);
  const int slot = blockIdx.x * kScoreThreads + threadIdx.x, lim = min(sq.old + sq.n, sq.len), nrows = sq.n * R;
  if (sq.n == 0 || slot >= lim || nrows > p.rows_over) return;
  const int pid = paged_page(a.c, b, slot / page);
  if (pid < 0) return;
  const bool fresh = slot >= sq.old;
  const int position = fresh ? (p.positions ? p.positions[sq.begin + slot - sq.old] : slot) : 0;
  const int64_t row0 = (int64_t)pid * G * page + slot % page, slots = (int64_t)a.c.max_pages * page;
  const float* src = a.score + ((int64_t)b * G * slots + slot) * ROWS;
#pragma unroll 4
  for (int g = 0; g < G; ++g) {
    float s[ROWS];
    const float* at = src + g * slots * ROWS;
    if constexpr (ROWS >= 4) {
#pragma unroll
      for (int i = 0; i < ROWS; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(at + i);
        s[i] = x.x; s[i + 1] = x.y; s[i + 2] = x.z; s[i + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) s[i] = at[i];
    }
    const int64_t row = row0 + (int64_t)g * page;
    float sum = fresh ? 0.f : p.weight[row];
    float add = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (i < nrows) {
        const float2 y = a.stat[(int64_t)(sq.begin + i / R) * a.b.H + g * R + i % R];
        add += fast_exp2(s[i] - y.x) * y.y;
      }
    p.weight[row] = sum + add;
    if (fresh) p.position[row] = position;
  }
}

cudaError_t scores_launch(const PagedWeighParams& p, cudaStream_t st) {
  const int64_t slots = (int64_t)p.a.c.max_pages * p.a.c.page;
  const dim3 grid((unsigned)((slots + kScoreThreads - 1) / kScoreThreads), p.a.b.B);
  switch (p.a.score_rows) {
    case 1: return launch_dependent(paged_weigh_scores_kernel<1>, grid, kScoreThreads, 0, st, p);
    case 2: return launch_dependent(paged_weigh_scores_kernel<2>, grid, kScoreThreads, 0, st, p);
    case 4: return launch_dependent(paged_weigh_scores_kernel<4>, grid, kScoreThreads, 0, st, p);
    case 8: return launch_dependent(paged_weigh_scores_kernel<8>, grid, kScoreThreads, 0, st, p);
    default: return cudaErrorInvalidValue;
  }
}

template <typename T, int KV>
cudaError_t weigh_launch(const PagedWeighParams& p, cudaStream_t st) {
  const PagedAttendParams& a = p.a;
  const int64_t slots = (int64_t)a.c.max_pages * a.c.page;
  const dim3 grid((unsigned)((slots + kSlots - 1) / kSlots), a.c.G, a.b.B);
  if (a.c.D == 128) return launch_dependent(paged_weigh_kernel<T, KV, 128>, grid, kSlots, 0, st, p);
  if (a.c.D == 64) return launch_dependent(paged_weigh_kernel<T, KV, 64>, grid, kSlots, 0, st, p);
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_paged_weigh(const PagedWeighParams& p, int dtype, int kv, cudaStream_t st) {
  if (p.a.score) {
    const cudaError_t e = scores_launch(p, st);
    if (e != cudaSuccess || (int64_t)p.a.b.max_tokens * (p.a.b.H / p.a.c.G) <= p.rows_over) return e;
  }
  if (dtype == kF16) return kv == kKvInt8 ? weigh_launch<__half, kKvInt8>(p, st) : weigh_launch<__half, kKvE4m3>(p, st);
  if (dtype == kBF16)
    return kv == kKvInt8 ? weigh_launch<__nv_bfloat16, kKvInt8>(p, st) : weigh_launch<__nv_bfloat16, kKvE4m3>(p, st);
  return cudaErrorInvalidValue;
}

}  // namespace spatten
