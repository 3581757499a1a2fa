// Attention over the paged 8-bit KV cache (spatten_paged_attend).
//
// One pass over the cache. The R = H / G query heads of a KV head and the n
// new tokens of a sequence make n R query rows that share the keys; a row tile
// is 8 or 16 of them. Per 16 keys, on the tensor cores with f16 operands (every
// int8 and e4m3 code is an f16) and fp32 sums:
//   S^T [16 keys x 8 rows]  = K codes . q'^T,
//   O^T [D x 8 rows]       += V codes^T . P^T.
// Both operands of the cache go from global memory into the fragments'
// registers: the order of the contracted dims (of S) and of the output dims (of
// O) is free, so each lane owns 16 consecutive bytes of a row, no shared memory
// is needed, and every byte is read once per row tile. P^T turns from the
// layout of S^T into that of an operand with one 8x8 transpose (movmatrix).
//
// Numerics:
//  * q' = q 2^e with the row's largest element in [2^14, 2^15): f16 then holds
//    bf16's range to 2^-39 of the row's largest element.
//  * s = (q' . codes) (sm_scale log2(e) 2^-e k_scale) in fp32, p = 2^(s - m) with
//    a reference m that follows the row's maximum (updated when it is exceeded
//    by more than 2^kSlack); l sums p in fp32.
//  * P is rounded to f16 for the second product (2^-11 of each weight), after
//    v_scale has gone into it: w = 2^(s + log2 v_scale - M), M a second reference
//    that follows max(s + log2 v_scale). A block with a tiny scale and all the weight
//    keeps its 11 bits beside blocks with large scales and no weight.
//
// Work split: the (sequence, KV head, row tile, 32-key tile) units are numbered
// and cut into equal ranges, one per CTA, over one wave of resident CTAs, from
// the lengths on the device: a ragged batch and one long sequence fill the GPU
// alike, and a captured launch follows the lengths it finds. The four warps of a
// CTA take turns on its tiles and join in shared memory; a (sequence, head, row
// tile) that a range's border cuts leaves (m, l, M, o) partials in the workspace,
// which a second kernel joins in a fixed order.
#include "kernels.h"
#include "paged_dev.cuh"

namespace spatten {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;        // keys per warp step: two 16-key blocks, each within one page
constexpr float kSlack = 8.f;    // p and w stay below 2^8
constexpr float kNoScale = -200.f;  // log2 of a scale of 0: below that of any float

// sequences whose prefix sums fit the shared memory
constexpr int kMaxBatch = 8192;

struct Workspace {
  int4* meta;   // [ctas]: parts of the row tile that starts in this CTA and is cut (0: none), b, g, row tile
  float4* ml;   // [2 ctas][rows] (m, l, M): slot 2 c: a tile begun before CTA c; 2 c + 1: one begun in it
  float* o;     // [2 ctas][rows][D]
};

template <int KV>
struct Codes;

// int8: x ^ 0x80 in the low byte of 0x6400 is the f16 1152 + x; the difference
// is exact. Bytes come out in the order (0, 2), (1, 3).
template <>
struct Codes<kKvInt8> {
  static constexpr int kPair = 2;  // distance of a pair's dims
  static SPATTEN_DEV uint32_t biased(uint32_t w) {
    const uint32_t u = (w & 0x00FF00FFu) ^ 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // a word of one row: the f16 pairs of its two k halves
  static SPATTEN_DEV void row(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = biased(w);
    hi = biased(w >> 8);
  }
  // words of two rows: the row pairs of dims 0 .. 3
  static SPATTEN_DEV void rows(uint32_t x, uint32_t y, uint32_t (&d)[4]) {
    const uint32_t t = __byte_perm(x, y, 0x5410), u = __byte_perm(x, y, 0x7632);
    d[0] = biased(t);
    d[1] = biased(t >> 8);
    d[2] = biased(u);
    d[3] = biased(u >> 8);
  }
};

template <>
struct Codes<kKvE4m3> {
  static constexpr int kPair = 1;
  static SPATTEN_DEV void row(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = e4m3x2_to_f16x2(w & 0xFFFFu);
    hi = e4m3x2_to_f16x2(w >> 16);
  }
  static SPATTEN_DEV void rows(uint32_t x, uint32_t y, uint32_t (&d)[4]) {
    const uint32_t t = __byte_perm(x, y, 0x5140), u = __byte_perm(x, y, 0x7362);
    row(t, d[0], d[1]);
    row(u, d[2], d[3]);
  }
};

SPATTEN_DEV uint4 ldg_stream16(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
SPATTEN_DEV uint2 ldg_stream8(const uint8_t* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

SPATTEN_DEV uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

SPATTEN_DEV float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }

// What takes an output by M to the result: 2^(M - m) / l, 0 for a row without a key.
SPATTEN_DEV float normaliser(float m, float l, float M) {
  return l == 0.f ? 0.f : exp2f(fminf(finite_or_0(M) - finite_or_0(m), 127.f)) / l;
}

// Row tiles of a sequence and 32-key tiles that its last row sees (one at
// least, so that rows without a key are written).
SPATTEN_DEV int row_tiles(const PagedSeq& s, int R, int rows) { return (int)(((int64_t)s.n * R + rows - 1) / rows); }
SPATTEN_DEV int key_tiles(const PagedSeq& s) { return max(1, (min(s.old + s.n, s.len) + kTile - 1) / kTile); }

template <int D, int NB>
struct Shape {
  static constexpr int kRows = 8 * NB;
  static constexpr int kOPad = D + 4;
  static constexpr int kCtas = NB == 1 ? 3 : 2;  // resident per SM: 170 / 255 registers per thread
  static constexpr size_t smem(int B) { return (size_t)(B + 1) * 8; }
};

// K words of a lane: [block][row gid, gid + 8][D / 16]; V words: [block][keys 2t, 2t+1, 2t+8, 2t+9][D / 32]
template <int D>
struct Tile {
  uint32_t k[2][2][D / 16];
  uint32_t v[2][4][D / 32];
};

template <int D>
SPATTEN_DEV void load_k(Tile<D>& t, int kb, const uint8_t* base, int gid, int tig) {
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const uint4 x = ldg_stream16(base + (gid + 8 * r) * D + 16 * (tig + 4 * j));
      t.k[kb][r][4 * j] = x.x; t.k[kb][r][4 * j + 1] = x.y;
      t.k[kb][r][4 * j + 2] = x.z; t.k[kb][r][4 * j + 3] = x.w;
    }
}

// rows at or behind `live` of the block read as zeros (their bytes may be anything)
template <int D>
SPATTEN_DEV void load_v(Tile<D>& t, int kb, const uint8_t* base, int gid, int tig, int live) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = 2 * tig + (r & 1) + 4 * (r & 2);
    const uint8_t* p = base + row * D + gid * (D / 8);
    if constexpr (D == 128) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (row < live) x = ldg_stream16(p);
      t.v[kb][r][0] = x.x; t.v[kb][r][1] = x.y; t.v[kb][r][2] = x.z; t.v[kb][r][3] = x.w;
    } else {
      uint2 x = make_uint2(0u, 0u);
      if (row < live) x = ldg_stream8(p);
      t.v[kb][r][0] = x.x; t.v[kb][r][1] = x.y;
    }
  }
}

template <int KV, int D, int NB>
__global__ void __launch_bounds__(32 * kWarps, Shape<D, NB>::kCtas)
paged_attend_kernel(const PagedAttendParams p, const Workspace ws, const bool bf16) {
  using SH = Shape<D, NB>;
  using C = Codes<KV>;
  constexpr int ROWS = SH::kRows, KS = D / 16, NT = 32 * kWarps;
  extern __shared__ __align__(16) long long pre[];  // [B + 1] units before each sequence
  __shared__ __align__(16) float sm_o[kWarps][ROWS][SH::kOPad];
  __shared__ float sm_m[kWarps][ROWS], sm_l[kWarps][ROWS], sm_M[kWarps][ROWS];
  __shared__ long long scan[kWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
  const int G = p.c.G, R = p.b.H / G, page = p.c.page;

  // prefix sums of the sequences' units
  long long carry = 0;
  if (tid == 0) pre[0] = 0;
  for (int base = 0; base < p.b.B; base += NT) {
    const int b = base + tid;
    long long x = 0;
    if (b < p.b.B) {
      const PagedSeq s = paged_seq(p.b, p.c, b);
      if (s.n > 0) x = (long long)G * row_tiles(s, R, ROWS) * key_tiles(s);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    long long before = carry;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      carry += scan[w];
    }
    if (b < p.b.B) pre[b + 1] = before + x;
    __syncthreads();
  }
  const long long U = carry;
  const int cta = blockIdx.x;
  const int ctas = (int)min((long long)gridDim.x, (U + kWarps - 1) / kWarps);  // a tile per warp at least
  int4 meta = make_int4(0, 0, 0, 0);
  if (cta >= ctas) {
    if (tid == 0) ws.meta[cta] = meta;
    return;
  }
  long long u = U * cta / ctas;
  const long long u1 = U * (cta + 1) / ctas;
  int b = 0;
  for (int hi = p.b.B; hi - b > 1;) {  // the sequence of unit u
    const int mid = (b + hi) >> 1;
    if (pre[mid] <= u) b = mid; else hi = mid;
  }

  while (u < u1) {
    while (pre[b + 1] <= u) ++b;
    const PagedSeq sq = paged_seq(p.b, p.c, b);
    const int KT = key_tiles(sq), RT = row_tiles(sq, R, ROWS);
    const long long local = u - pre[b];
    const int g = (int)(local / ((long long)RT * KT));
    const int rem = (int)(local - (long long)g * RT * KT), rt = rem / KT, t0 = rem % KT;
    const int t1 = (int)min((long long)KT, t0 + (u1 - u));
    const int nrows = sq.n * R, r0 = rt * ROWS;
    // slots that the tile's last and first row see
    const int lim_max = min(sq.old + min((r0 + ROWS - 1) / R, sq.n - 1) + 1, sq.len);
    const int lim_min = min(sq.old + r0 / R + 1, sq.len);
    const int t_end = min(t1, (max(lim_max, 0) + kTile - 1) / kTile);

    // queries: row gid of each 8-row block, all dims of it in the four lanes of gid
    uint32_t qf[NB][KS][2];
    float cq[NB][2], m[NB][2], M[NB][2], l[NB][2];
    int lim[NB][2];
    float o[NB][KS][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = r0 + nb * 8 + gid;
      const bool live = r < nrows;
      const int64_t at = live ? (int64_t)(sq.begin + r / R) * p.q_st + (int64_t)(g * R + r % R) * p.q_sh : 0;
      const uint16_t* qp = static_cast<const uint16_t*>(p.q) + at;
      uint2 raw[KS];
      float top = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        raw[s] = live ? __ldg(reinterpret_cast<const uint2*>(qp + 16 * (tig + 4 * (s / 4)) + 4 * (s % 4)))
                      : make_uint2(0u, 0u);
        const uint32_t w[2] = {raw[s].x, raw[s].y};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float2 f;
          if (bf16) f = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
          else f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e: top in [2^14, 2^15), e at most 126
      const int e = top > 0.f ? 14 - max((int)(__float_as_uint(top) >> 23) - 127, -112) : 0;
      const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint32_t w[2] = {raw[s].x, raw[s].y};
        float f[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float2 x;
          if (bf16) x = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
          else x = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          f[2 * j] = x.x * up;
          f[2 * j + 1] = x.y * up;
        }
        // the pairs that Codes::row makes of a word
        qf[nb][s][0] = pack2<__half>(f[0], f[C::kPair]);
        qf[nb][s][1] = pack2<__half>(f[3 - C::kPair], f[3]);
      }
      const float c = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // this lane's rows of the products: 2 tig, 2 tig + 1
        cq[nb][j] = __shfl_sync(0xffffffffu, c, (2 * tig + j) * 4);
        lim[nb][j] = min(sq.old + (r0 + nb * 8 + 2 * tig + j) / R + 1, sq.len);
        m[nb][j] = M[nb][j] = -INFINITY;
        l[nb][j] = 0.f;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[nb][s][j] = 0.f;
    }

    // this warp's tiles t0 + warp, + 4, ..: lane i keeps the page and scales of
    // the 16-key block i & 1 of tile i >> 1 of the 16 tiles at hand, and the
    // page-table entry of the 16 tiles after them
    const int nt = t_end > t0 + warp ? (t_end - t0 - warp + kWarps - 1) / kWarps : 0;
    auto block_slot = [&](int j) { return (t0 + warp + kWarps * j) * kTile; };
    auto entry = [&](int j) {
      const int slot = block_slot(j + (lane >> 1)) + 16 * (lane & 1);
      return slot < lim_max ? paged_page(p.c, b, slot / page) : -1;
    };
    int pid_l = -1, pid_n = -1;
    float ks_l = 0.f, vs_l = 0.f;
    auto scales = [&]() {
      const int64_t blk = (int64_t)max(pid_l, 0) * G + g;
      ks_l = pid_l >= 0 ? __ldg(p.c.k_scale + blk) : 0.f;
      vs_l = pid_l >= 0 ? __ldg(p.c.v_scale + blk) : 0.f;
    };
    Tile<D> tile;
    int pid[2] = {-1, -1};  // of the tile in registers (its V part may still be the one before)
    auto at = [&](const uint8_t* x, int which, int slot) {
      return x + (((int64_t)max(which, 0) * G + g) * page + (slot & (page - 1))) * D;
    };
    if (nt > 0) {
      pid_l = entry(0);
      pid_n = entry(16);
      scales();
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        pid[kb] = __shfl_sync(0xffffffffu, pid_l, kb);
        const int slot = block_slot(0) + 16 * kb;
        if (pid[kb] >= 0) load_k<D>(tile, kb, at(p.c.k, pid[kb], slot), gid, tig);
        load_v<D>(tile, kb, at(p.c.v, pid[kb], slot), gid, tig, pid[kb] >= 0 ? lim_max - slot : 0);
      }
    }
    for (int j = 0; j < nt; ++j) {
      const int slot0 = block_slot(j);
      if ((j & 15) == 0) vs_l = vs_l > 0.f ? fmaxf(log2f(vs_l), kNoScale) : kNoScale;  // from here on: its log2
      float ks[2], lv[2];
      const int now[2] = {pid[0], pid[1]};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        ks[kb] = __shfl_sync(0xffffffffu, ks_l, 2 * (j & 15) + kb);
        lv[kb] = __shfl_sync(0xffffffffu, vs_l, 2 * (j & 15) + kb);
      }
      // scores
      float s[2][NB][4];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kb][nb][i] = 0.f;
        if (now[kb] < 0) continue;  // warp-uniform: no memory, masked below
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t a[4];
          C::row(tile.k[kb][0][k], a[0], a[2]);
          C::row(tile.k[kb][1][k], a[1], a[3]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma_16816<__half>(s[kb][nb], a, qf[nb][k][0], qf[nb][k][1]);
        }
      }
      // the next tile's keys on their way
      int next[2] = {-1, -1};
      const int slot1 = block_slot(j + 1);
      if (j + 1 < nt) {
        if (((j + 1) & 15) == 0) {
          pid_l = pid_n;
          pid_n = entry(j + 17);
          scales();
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          next[kb] = __shfl_sync(0xffffffffu, pid_l, 2 * ((j + 1) & 15) + kb);
          if (next[kb] >= 0) load_k<D>(tile, kb, at(p.c.k, next[kb], slot1 + 16 * kb), gid, tig);
        }
      }
      // p = 2^(s - m), and w = 2^(s + log2 v_scale - M)
      const bool masked = slot0 + kTile > lim_min || now[0] < 0 || now[1] < 0;
      float top[NB][2], topw[NB][2];  // largest s, and s + log2 v_scale, of this lane
      bool up = false;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float t[2];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            const float f = cq[nb][c] * ks[kb];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float& x = s[kb][nb][2 * i + c];
              x *= f;
              if (masked && (now[kb] < 0 || slot0 + 16 * kb + gid + 8 * i >= lim[nb][c])) x = -INFINITY;
            }
            t[kb] = fmaxf(s[kb][nb][c], s[kb][nb][2 + c]);
          }
          top[nb][c] = fmaxf(t[0], t[1]);
          topw[nb][c] = fmaxf(t[0] + lv[0], t[1] + lv[1]);
          up |= top[nb][c] > m[nb][c] + kSlack || topw[nb][c] > M[nb][c] + kSlack;
        }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = top[nb][c], y = topw[nb][c];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
              y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
            }
            const float mn = fmaxf(m[nb][c], x), Mn = fmaxf(M[nb][c], y);
            l[nb][c] *= fast_exp2(m[nb][c] - finite_or_0(mn));
            const float f = fast_exp2(M[nb][c] - finite_or_0(Mn));
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              o[nb][k][c] *= f;
              o[nb][k][2 + c] *= f;
            }
            m[nb][c] = mn;
            M[nb][c] = Mn;
          }
      }
      uint32_t pf[2][NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float mf[2], Mf[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mf[c] = finite_or_0(m[nb][c]);
          Mf[c] = finite_or_0(M[nb][c]);
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float s0 = s[kb][nb][2 * i], s1 = s[kb][nb][2 * i + 1];
            l[nb][0] += fast_exp2(s0 - mf[0]);
            l[nb][1] += fast_exp2(s1 - mf[1]);
            pf[kb][nb][i] = transpose8x8(
                pack2<__half>(fast_exp2(s0 + (lv[kb] - Mf[0])), fast_exp2(s1 + (lv[kb] - Mf[1]))));
          }
      }
      // values
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          uint32_t lo[4], hi[4];
          C::rows(tile.v[kb][0][w], tile.v[kb][1][w], lo);
          C::rows(tile.v[kb][2][w], tile.v[kb][3][w], hi);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a[4] = {lo[2 * h], lo[2 * h + 1], hi[2 * h], hi[2 * h + 1]};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma_16816<__half>(o[nb][2 * w + h], a, pf[kb][nb][0], pf[kb][nb][1]);
          }
        }
      // and the next tile's values
      if (j + 1 < nt) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          pid[kb] = next[kb];
          const int slot = slot1 + 16 * kb;
          load_v<D>(tile, kb, at(p.c.v, pid[kb], slot), gid, tig, pid[kb] >= 0 ? lim_max - slot : 0);
        }
      }
    }

    // the warps join, sums by m and outputs by M
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = nb * 8 + 2 * tig + c;
        float sum = l[nb][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        float4* dst = reinterpret_cast<float4*>(&sm_o[warp][row][gid * (D / 8)]);
#pragma unroll
        for (int k = 0; k < KS; k += 2)
          dst[k / 2] = make_float4(o[nb][k][c], o[nb][k][2 + c], o[nb][k + 1][c], o[nb][k + 1][2 + c]);
        if (gid == 0) {
          sm_m[warp][row] = m[nb][c];
          sm_l[warp][row] = sum;
          sm_M[warp][row] = M[nb][c];
        }
      }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == KT;
    const int slot = 2 * cta + (t0 == 0 ? 1 : 0);
    for (int i = tid; i < ROWS * (D / 4); i += NT) {
      const int row = i / (D / 4), d = (i % (D / 4)) * 4, r = r0 + row;
      if (r >= nrows) break;
      float mm = -INFINITY, MM = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        mm = fmaxf(mm, sm_m[w][row]);
        MM = fmaxf(MM, sm_M[w][row]);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = fast_exp2(sm_M[w][row] - finite_or_0(MM));
        const float4 x = *reinterpret_cast<const float4*>(&sm_o[w][row][d]);
        ll += sm_l[w][row] * fast_exp2(sm_m[w][row] - finite_or_0(mm));
        acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
      }
      if (whole) {
        const float inv = normaliser(mm, ll, MM);
        uint16_t* op = static_cast<uint16_t*>(p.out) + (int64_t)(sq.begin + r / R) * p.o_st +
                       (int64_t)(g * R + r % R) * p.o_sh + d;
        uint2 v;
        v.x = bf16 ? pack2<__nv_bfloat16>(acc.x * inv, acc.y * inv) : pack2<__half>(acc.x * inv, acc.y * inv);
        v.y = bf16 ? pack2<__nv_bfloat16>(acc.z * inv, acc.w * inv) : pack2<__half>(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(op) = v;
      } else {
        *reinterpret_cast<float4*>(ws.o + ((int64_t)slot * ROWS + row) * D + d) = acc;
        if (d == 0) ws.ml[(int64_t)slot * ROWS + row] = make_float4(mm, ll, MM, 0.f);
      }
    }
    if (t0 == 0 && !whole) {  // cut: the CTAs up to that of its last unit hold a part each
      const long long end = u + KT;
      meta = make_int4((int)((end * ctas + U - 1) / U) - cta, b, g, rt);
    }
    __syncthreads();
    u += t1 - t0;
  }
  if (tid == 0) ws.meta[cta] = meta;
}

// Joins the row tile that starts in CTA blockIdx.x and is cut: its parts are
// slot 2 c + 1 of that CTA and slot 2 c of the following ones. A warp per row.
template <int D, int ROWS>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttendParams p, const Workspace ws, const bool bf16) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int E = D / 32;
  const int c0 = blockIdx.x, lane = threadIdx.x & 31;
  const int4 meta = ws.meta[c0];
  if (meta.x <= 1) return;
  const int parts = meta.x, g = meta.z, R = p.b.H / p.c.G;
  const PagedSeq sq = paged_seq(p.b, p.c, meta.y);
  for (int row = threadIdx.x >> 5; row < ROWS; row += 8) {
    const int r = meta.w * ROWS + row;
    if (r >= sq.n * R) return;
    auto at = [&](int i) { return ((int64_t)(i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * ROWS + row); };
    float mm = -INFINITY, MM = -INFINITY;
    for (int i = lane; i < parts; i += 32) {
      const float4 x = ws.ml[at(i)];
      mm = fmaxf(mm, x.x);
      MM = fmaxf(MM, x.z);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
      MM = fmaxf(MM, __shfl_xor_sync(0xffffffffu, MM, d));
    }
    float l = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 32) {
      float f = 0.f;
      if (i0 + lane < parts) {
        const float4 x = ws.ml[at(i0 + lane)];
        f = fast_exp2(x.z - finite_or_0(MM));
        l += x.y * fast_exp2(x.x - finite_or_0(mm));
      }
      const int n = min(32, parts - i0);
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float w = __shfl_sync(0xffffffffu, f, i);
        const float* src = ws.o + at(i0 + i) * D + lane * E;
        if constexpr (E == 4) {
          const float4 x = *reinterpret_cast<const float4*>(src);
          acc[0] += x.x * w; acc[1] += x.y * w; acc[2] += x.z * w; acc[3] += x.w * w;
        } else {
          const float2 x = *reinterpret_cast<const float2*>(src);
          acc[0] += x.x * w; acc[1] += x.y * w;
        }
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    const float inv = normaliser(mm, l, MM);
    uint16_t* op = static_cast<uint16_t*>(p.out) + (int64_t)(sq.begin + r / R) * p.o_st +
                   (int64_t)(g * R + r % R) * p.o_sh + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2)
      *reinterpret_cast<uint32_t*>(op + e) =
          bf16 ? pack2<__nv_bfloat16>(acc[e] * inv, acc[e + 1] * inv) : pack2<__half>(acc[e] * inv, acc[e + 1] * inv);
  }
}

// Eight query rows per pass where that covers a sequence's rows (the register
// tile of 16 has room for half the bytes in flight), else sixteen.
int row_block(const PagedAttendParams& p) { return (int64_t)p.b.max_tokens * (p.b.H / p.c.G) <= 8 ? 8 : 16; }

int grid_ctas(const PagedAttendParams& p, int n_sm) { return n_sm * (row_block(p) == 8 ? 3 : 2); }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

template <int KV, int D, int NB>
cudaError_t attend_launch(const PagedAttendParams& p, bool bf16, const Workspace& ws, int ctas, cudaStream_t st) {
  using SH = Shape<D, NB>;
  const size_t smem = SH::smem(p.b.B);
  cudaError_t e = cudaFuncSetAttribute(paged_attend_kernel<KV, D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)SH::smem(kMaxBatch));
  if (e != cudaSuccess) return e;
  paged_attend_kernel<KV, D, NB><<<ctas, 32 * kWarps, smem, st>>>(p, ws, bf16);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // scheduled while the first kernel drains; it waits for its results itself
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<D, SH::kRows>, p, ws, bf16);
}

template <int KV, int D>
cudaError_t attend_rows(const PagedAttendParams& p, bool bf16, const Workspace& ws, int ctas, cudaStream_t st) {
  return row_block(p) == 8 ? attend_launch<KV, D, 1>(p, bf16, ws, ctas, st)
                           : attend_launch<KV, D, 2>(p, bf16, ws, ctas, st);
}

template <int KV>
cudaError_t attend_dim(const PagedAttendParams& p, bool bf16, const Workspace& ws, int ctas, cudaStream_t st) {
  if (p.c.D == 128) return attend_rows<KV, 128>(p, bf16, ws, ctas, st);
  if (p.c.D == 64) return attend_rows<KV, 64>(p, bf16, ws, ctas, st);
  return cudaErrorInvalidValue;
}

}  // namespace

int paged_attend_max_batch() { return kMaxBatch; }

size_t paged_attend_workspace(const PagedAttendParams& p, int n_sm) {
  const size_t ctas = grid_ctas(p, n_sm), rows = row_block(p);
  return align256(ctas * sizeof(int4)) + align256(2 * ctas * rows * sizeof(float4)) +
         align256(2 * ctas * rows * p.c.D * sizeof(float));
}

cudaError_t launch_paged_attend(const PagedAttendParams& p, int dtype, int kv, void* ws, int n_sm, cudaStream_t st) {
  if (dtype != kF16 && dtype != kBF16) return cudaErrorInvalidValue;
  const int ctas = grid_ctas(p, n_sm), rows = row_block(p);
  uint8_t* w = static_cast<uint8_t*>(ws);
  Workspace s;
  s.meta = reinterpret_cast<int4*>(w);
  w += align256(ctas * sizeof(int4));
  s.ml = reinterpret_cast<float4*>(w);
  w += align256((size_t)2 * ctas * rows * sizeof(float4));
  s.o = reinterpret_cast<float*>(w);
  const bool bf16 = dtype == kBF16;
  return kv == kKvInt8 ? attend_dim<kKvInt8>(p, bf16, s, ctas, st) : attend_dim<kKvE4m3>(p, bf16, s, ctas, st);
}

}  // namespace spatten
