// Host-side declarations of the operators over a paged cache (paged.cu, sm100_paged.cu, sm100_latent.cu) and of keys that share columns.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>
#include "common.cuh"

namespace ab200 {

struct BlockTables {
  int32_t batch, page, width;
  int64_t total, table_stride, num_free;
  int32_t* table;
  const int32_t *lengths, *new_tokens, *free_pages, *taken;
  int64_t* slots;
  int32_t *cu_seqlens, *new_lengths, *taken_out;
};

struct PagedWrite {
  int64_t tokens, slots_total;       // slots of the cache: what lies outside them is not written
  int32_t page, heads, dk, dv;       // dv 0: keys alone
  const void *k, *v;
  void *k_cache, *v_cache;
  int64_t sk[2], sv[2];              // strides of tokens and heads
  int64_t ck[3], cv[3];              // strides of pages, slots and heads
  const int64_t* slots;
  int32_t vec;                       // bytes that every row allows at a time
};

// Attention of the last queries of each sequence over pages.  Sequence z has the first lengths[z] keys of its table's pages; its
// query m stands at position lengths[z] - queries + m.
struct PagedAttn {
  View4 q, out;                      // (B, Hq, Sq, D)
  View4 k, v;                        // (pages, page, Hk, D)
  const int32_t* table;
  int64_t table_stride;
  int32_t width, page, num_pages;
  const int32_t *lengths, *query_lengths;
  float* lse;                        // (B * Hq, Sq), or null
  int32_t batch, hq, hk, group, sq, dqk, dvo;
  float qk_scale;                    // sm_scale * log2(e)
  int32_t window, sinks;             // window INT32_MAX: none
  int32_t max_len;                   // what the table has room for
  // How the call is cut (plan_paged, paged_split.cuh): into units -- (sequence, kv head, chunk of `rows` query rows) -- and tiles of 2^tile_log keys, for `ctas`
  // CTAs, min_tiles a CTA at least, a unit counted as `extra` tiles more than it has; `lanes` chunks side by side (a divisor of the chunks, and of the CTAs).
  // box: slots of a tile copy.  slice: sequences of a launch, fewer than all where their tables have room for more tiles than are counted.
  int32_t kind, ctas, lanes, rows, chunks, tile_log, min_tiles, extra, box, slice;
  int32_t q_tiles;                   // latent attention: the queries come as tile copies
  unsigned int* status;              // the word in which a kernel records a wait that ran out (null: the general kernel has none)
  float* partial;                    // two partial results a CTA: of the unit that it starts with, of the one that it ends with
  uint32_t wait_limit_kcycles;
  int32_t drop_copy;
};

enum PagedKind : int { kPagedGeneral = 1, kPagedSplit = 2, kPagedLatent = 3 };

// Which tokens of keys are of a sequence (Params' fields of the same names), of no more than max_sk keys.
struct KeyTokens {
  int32_t varlen_mode, batch, max_sk;
  const int32_t *cu_k, *ss_k;
};
struct SharedColumns {
  View4 k, shared, out;              // (B, H, S, dn), (B, 1, S, dr), (B, H, S, dn + dr)
  KeyTokens tokens;                  // the gradient's: rows of no sequence are zero
};

cudaError_t launch_block_tables(const BlockTables& a, cudaStream_t st);
cudaError_t launch_paged_write(int dtype, const PagedWrite& a, cudaStream_t st);
// Chooses the kernel and how the call is cut for `sms` SMs; returns the floats of workspace it needs, or -kPagedTooLarge: a table row with room for more tiles than
// are counted.
constexpr int64_t kPagedTooLarge = 1;
int64_t plan_paged(int dtype, PagedAttn& a, int sms);
cudaError_t launch_paged(int dtype, PagedAttn& a, cudaStream_t st);
// The tensor-core kernels: whether one takes the call, and if so how it cuts it (all but ctas' bound and the workspace); and its launch.
bool plan_paged_split(int dtype, PagedAttn& a, int sms);
cudaError_t launch_paged_split(int dtype, PagedAttn& a, cudaStream_t st);
bool plan_paged_latent(int dtype, PagedAttn& a, int sms);
cudaError_t launch_paged_latent(int dtype, PagedAttn& a, cudaStream_t st);
// The status word of the current device (sm100_paged.cu), as sm100_fwd_status has it.
cudaError_t paged_status_word(unsigned int** word, int* dev, bool* remember);
unsigned int sm100_paged_status(bool reset);
cudaError_t launch_join_columns(int dtype, const SharedColumns& a, cudaStream_t st);
cudaError_t launch_sum_columns(int dtype, const SharedColumns& a, cudaStream_t st);      // shared = sum over heads of out's last columns

// ... from dK's last columns in 32 bits, (batch, kv heads, tokens, columns).
cudaError_t launch_sum_tail(int dtype, const SharedColumns& a, const float* tail, int heads, cudaStream_t st);

}  // namespace ab200
