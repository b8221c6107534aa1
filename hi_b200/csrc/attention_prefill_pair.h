// The tcgen05 prefill attention of plain softmax rows, two query tiles a block (attention_prefill_pair.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

struct PrefillPairArgs {
  const int* block_table;
  const int* cu_seqlens;
  const int* positions;
  __nv_bfloat16* out;
  int* status;
  int table_stride, nh, nkv, page_size, chunk, window, skip_single, box_rows;
  float scale_log2;          // softmax scale * log2(e)
  // With key_splits > 1 that many blocks share the key tiles of every pair of items; a block leaves its rows unnormalised in
  // part_acc [row][split][head_dim] with (maximum, sum) in part_ml [row][split][2], and hb_attention_merge combines them.
  int key_splits;
  float* part_acc;
  float* part_ml;
  int sink;                  // 1: the denominator has one more term, e^0, or e^sink_values[head]
  const float* sink_values;
  // not null: requests and kv heads have forms of their own (four_bit_cache.cu). form[seq][kv head]: what the values have been divided by, and
  // 1 for q, k and v in float16; q_scale[token][head]: a row's own scale_log2, a power of two where scores may be large, so that their maximum
  // times it is not rounded
  const float2* form;
  const float* q_scale;
};

// What rows held in float16 add to their weights' exponents: a weight is 2^(score - m + RAISE), at most 2^(8 + RAISE) where the maximum m is
// followed within 2^8, which float16 holds (65,504), as it then holds weights down to 2^-(24 + RAISE) of one at m. (Without, keys of 2^-26 of the
// largest weight were lost from the values' sum and not from the weights': 131,072 of them are 2^-9 of it.)
constexpr float RAISE = 7.f;

// head_dim 64 or 128; HB_ERR_UNSUPPORTED for others
int hb_prefill_pair_launch(const void* q, const void* k_pages, const void* v_pages, const PrefillPairArgs& a, int n_tokens,
                           long long pool_rows, int n_seqs, int max_new, int hd, cudaStream_t stream);
