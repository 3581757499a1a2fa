// Trees of drafted tokens (spatten_paged_tree): which of its sequence's new
// tokens each of them sees, as bits, and its position.
//
//   sees(i) = {i} and sees(parent(i)),  position(i) = old + depth(i)
//
// A parent comes before its child (another value makes the token a child of the
// cached ones), so a thread per token follows its chain downwards through the
// parents in shared memory and finishes a word of bits when the chain leaves it.
// Bound by latency (lengths, parents, a step of the chain per level): one tree of 26
// tokens 1.8 us of device time, 64 trees of up to 64 4.4 to 4.6 us. A CTA per sequence, so that
// its parents are read once; one call serves all layers of a step.
#include "kernels.h"
#include "paged_dev.cuh"

namespace spatten {
namespace {

constexpr int kTreeThreads = 256;

__global__ void __launch_bounds__(kTreeThreads) paged_tree_kernel(const PagedTreeParams p) {
  __shared__ int up[kTreeTokens];
  grid_dependents();
  grid_wait();
  const int b = blockIdx.x, tid = threadIdx.x;
  const int lo = *(p.b.cu + b), hi = *(p.b.cu + b + 1), len = min(max(*(p.b.lens + b), 0), 1 << 30);
  const int rows = lo >= 0 && lo <= hi && hi <= p.b.T ? hi - lo : 0, n = min(rows, p.b.max_tokens);
  for (int i = tid; i < n; i += kTreeThreads) {
    const int a = *(p.parents + lo + i);
    up[i] = a >= 0 && a < i ? a : -1;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kTreeThreads) {
    uint32_t* out = p.tree + (int64_t)(lo + i) * p.tree_st;
    int word = p.words - 1, depth = -1;
    uint32_t bits = 0u;
    for (int a = i; a >= 0; a = up[a], ++depth) {
      for (; word > a >> 5; --word) {
        out[word] = bits;
        bits = 0u;
      }
      bits |= 1u << (a & 31);
    }
    for (; word >= 0; --word) {
      out[word] = bits;
      bits = 0u;
    }
    if (p.positions) p.positions[lo + i] = len - rows + depth;
  }
}

}  // namespace

cudaError_t launch_paged_tree(const PagedTreeParams& p, cudaStream_t st) {
  return launch_dependent(paged_tree_kernel, dim3(p.b.B), kTreeThreads, 0, st, p);
}

}  // namespace spatten
