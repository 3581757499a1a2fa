// Paged 8-bit KV cache: append (paged.cu), read back (paged.cu) and attention
// over it (paged_attend.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace spatten {

enum KvType : int { kKvInt8 = 0, kKvE4m3 = 1 };

struct PagedCache {
  int P, page, G, D;        // pages, tokens per page, KV heads, head dim
  int max_pages;            // page-table columns
  uint8_t* k;               // [P, G, page, D] codes
  uint8_t* v;
  float* k_scale;           // [P, G]
  float* v_scale;
  const int32_t* table;     // [B, max_pages], row stride table_st
  int64_t table_st;
};

// The new tokens of a batch, packed.
struct PagedBatch {
  int B, H, T, max_tokens;
  const int32_t* cu;        // [B + 1]
  const int32_t* lens;      // [B] tokens held, the new ones included
};

struct PagedAppendParams {
  PagedCache c;
  PagedBatch b;
  const void* q;            // or null
  int64_t q_st, q_sh;
  const void* k;
  int64_t k_st, k_sh;
  const void* v;
  int64_t v_st, v_sh;
  void* q_out;
  int64_t qo_st, qo_sh;
  const void* wq;           // or null
  const void* wk;
  float eps;
  const void* cos;          // or null
  const void* sin;
  bool cs_f32;
  int cs_rows;
  int64_t cs_st;
  const int32_t* positions; // or null
};

struct PagedAttendParams {
  PagedCache c;
  PagedBatch b;
  const void* q;
  int64_t q_st, q_sh;
  void* out;
  int64_t o_st, o_sh;
  float scale_log2;         // sm_scale * log2(e)
  // the launch serves sequences with more than rows_over and at most rows_upto
  // query rows per KV head
  int64_t rows_over, rows_upto;
};

struct PagedReadParams {
  PagedCache c;
  int B, N;
  const int32_t* lens;
  const int64_t* idx;       // or null
  int64_t idx_st;
  void* k_out;
  void* v_out;
};

cudaError_t launch_paged_append(const PagedAppendParams& p, int dtype, int kv, cudaStream_t st);
cudaError_t launch_paged_read(const PagedReadParams& p, int dtype, int kv, cudaStream_t st);
int paged_attend_max_batch();  // sequences of one call
bool paged_attend_fits(const PagedAttendParams& p);  // units of work count in 32 bits
size_t paged_attend_workspace(const PagedAttendParams& p, int n_sm);
// the tcgen05 path (paged_attend_tc.cu), for many query rows per KV head
constexpr int kTcRows = 64;  // it takes sequences with more rows than this
bool paged_attend_tc_takes(const PagedAttendParams& p);
size_t paged_attend_tc_workspace(const PagedAttendParams& p, int n_sm);
cudaError_t launch_paged_attend_tc(const PagedAttendParams& p, int dtype, int kv, void* ws, int n_sm,
                                   cudaStream_t st);
cudaError_t read_paged_device_error(unsigned int* code, bool reset);
cudaError_t launch_paged_attend(const PagedAttendParams& p, int dtype, int kv, void* ws, int n_sm,
                                cudaStream_t st);

}  // namespace spatten
