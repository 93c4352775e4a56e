// Launch functions of the paged key/value cache (paged_append.cu, paged_attention.cu), called by their PyTorch
// side (paged_torch.cpp), which checks the arguments. Nothing here needs PyTorch.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace me {

// A batch of sequences in the cache and their new tokens, which are packed: sequence b has the tokens
// cu[b] .. cu[b + 1] - 1, its last ones, and lens[b] tokens in all.
struct PagedBatch {
  const int *cu, *lens;
  const int* table;      // [seqs, width] page of each run of `page` positions
  int64_t table_stride;  // elements between its rows
  int width, seqs, tokens;
};

// Pages [pages, heads, page, dim] of keys and of values (bf16); a page's elements are contiguous, pages any multiple of
// 8 elements apart.
struct PagedCache {
  void *k, *v;
  int64_t k_stride, v_stride;
  int pages, heads, page, dim;
};

struct AppendArgs {
  PagedBatch batch;
  PagedCache cache;
  const void* qkv;       // [tokens, (q heads + (1 | 2) heads) dim] bf16
  int64_t qkv_stride;
  const float *q_w, *k_w, *inv_freq;
  void* q;               // [tokens, q heads, dim]
  int q_heads;
  bool kv_shared;
  float eps;
};
void launch_paged_append(const AppendArgs& a, int sms, cudaStream_t stream);

struct PagedAttentionArgs {
  PagedBatch batch;
  PagedCache cache;
  const void* q;         // [tokens, q heads, dim] bf16, strides in elements
  int64_t q_token, q_head;
  void* o;               // the same with its own strides
  int64_t o_token, o_head;
  float* lse;            // [q heads, tokens]
  int q_heads, window;   // window 0: none
  float scale;
  bool clear_rest;       // rows of no sequence: zeros in o (else left as they are; lse is -inf either way)
  int max_q;             // the longest run of new tokens, as far as the caller knows
};
// Bytes of workspace that the call needs (16-byte aligned), and the call; what is wrong, if anything is.
int64_t paged_attention_workspace(const PagedAttentionArgs& a, int sms);
const char* launch_paged_attention(const PagedAttentionArgs& a, void* workspace, int sms, cudaStream_t stream);

// Its part for sequences with more than `least_rows` rows (new tokens times query heads of a key head): paged_tiles.cu.
int64_t paged_tiles_workspace(const PagedAttentionArgs& a);
const char* launch_paged_tiles(const PagedAttentionArgs& a, int least_rows, void* workspace, cudaStream_t stream);
// On the current device: blocks in which a wait ran out since the process began, and where the last of them waited. Waits for `stream`, which is not
// being captured.
cudaError_t paged_waits(int (&words)[2], cudaStream_t stream);

}  // namespace me
