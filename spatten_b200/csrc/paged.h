// Paged 8-bit KV cache: append (paged.cu), read back (paged.cu), attention over
// it (paged_attend.cu, paged_attend_tc.cu), the weights that it gives the cached
// tokens (paged_weigh.cu), trees of drafted tokens (paged_tree.cu), and tokens that
// leave the cache (paged_evict.cu).
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
  // beside the causal form:
  const uint32_t* tree = nullptr;  // or null: bits of the new tokens that a row sees, [T, words]
  int64_t tree_st = 0;
  int words = 0;
  float2* stat = nullptr;          // or null: [T, H] reference m of a row's exponentials, 1 / their sum
  // or null: scores (log2) of sequences of at most score_rows query rows per KV
  // head, [slot_place][score_rows], where an unmasked place's page has memory
  float* score = nullptr;
  int score_rows = 0;
  bool by_pool = false;            // see slot_places
};
constexpr int kScoreRows = 32;   // at most

// What a call keeps for each of its slots (of which sequences share none) lies by
// sequence and slot, [B, G, slots], or like the pool, [P, G, page]: whichever is smaller.
inline int64_t slot_places(const PagedAttendParams& p, bool by_pool) {
  return by_pool ? (int64_t)p.c.P * p.c.G * p.c.page : (int64_t)p.b.B * p.c.G * p.c.max_pages * p.c.page;
}

// The weights that a call's rows give the cached tokens (after the attention).
struct PagedWeighParams {
  PagedAttendParams a;      // its stat is read
  float* weight;            // [P, G, page]
  int32_t* position;        // [P, G, page]
  const int32_t* positions; // or null: [T]
  int rows_over;            // sequences of at most as many rows have their scores kept
};

struct PagedTreeParams {
  PagedBatch b;
  const int32_t* parents;   // [T]
  uint32_t* tree;           // [T, words]
  int64_t tree_st;
  int words;
  int32_t* positions;       // or null: [T]
};

struct PagedEvictParams {
  PagedCache c;
  int B;
  const int32_t* lens;
  float* weight;
  int32_t* position;
  int keep, recent;
  bool per_head;
  int32_t* new_lens;
};

struct PagedKeepParams {
  PagedCache c;
  PagedBatch b;
  const int32_t* accepted;  // [B, A], row stride accepted_st
  int64_t accepted_st;
  int A;
  float* weight;            // or null
  int32_t* position;
  int32_t* new_lens;
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
constexpr int kTcRows = 64;       // it takes sequences with more rows than this,
constexpr int kTcRowsAlike = 48;  // or this where all have as many
bool paged_attend_tc_takes(const PagedAttendParams& p);
size_t paged_attend_tc_workspace(const PagedAttendParams& p, int n_sm);
cudaError_t launch_paged_attend_tc(const PagedAttendParams& p, int dtype, int kv, void* ws, int n_sm,
                                   cudaStream_t st);
cudaError_t read_paged_device_error(unsigned int* code, bool reset);
cudaError_t launch_paged_attend(const PagedAttendParams& p, int dtype, int kv, void* ws, int n_sm,
                                cudaStream_t st);
int paged_attend_score_rows(const PagedAttendParams& p);  // scores kept per slot; 0: none
size_t paged_weigh_workspace(const PagedWeighParams& p);
cudaError_t launch_paged_weigh(const PagedWeighParams& p, int dtype, int kv, void* ws, int n_sm, cudaStream_t st);
cudaError_t read_paged_weigh_error(unsigned int* code, bool reset);
constexpr int kTreeTokens = 1024;  // new tokens of a sequence whose tree is laid out
cudaError_t launch_paged_tree(const PagedTreeParams& p, cudaStream_t st);
constexpr int kEvictSlots = 1 << 20;  // slots of a sequence that is chosen from
size_t paged_evict_workspace(const PagedEvictParams& p);
cudaError_t launch_paged_evict(const PagedEvictParams& p, int kv, void* ws, int n_sm, cudaStream_t st);
cudaError_t launch_paged_keep(const PagedKeepParams& p, int kv, cudaStream_t st);

}  // namespace spatten
