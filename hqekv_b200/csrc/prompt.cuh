// What prompt.cu offers to decode.cu, and the arguments of its kernels.
#pragma once

#include <cuda_bf16.h>

#include <cuda.h>

#include "common.cuh"

namespace hqkv {

struct PromptArgs {
  const void *q, *k, *v, *pk, *pv;                  // element (token, head, channel) at token * stride + head * stride + channel
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, pk_token, pk_head, pv_token, pv_head;
  const int *q_starts, *k_starts;                   // [n_seqs + 1]
  int n_seqs, total_q, total_k, prefix_len, nh_q, nh_kv;
  int group, groups, groups_per_kv;                 // query heads of a kv head that share a row tile; such groups
  int row_shift, block_shift;                       // log2 of the tokens of a row tile, of a block (one or two row tiles)
  int per_share, shares;                            // tiles of keys per share of a block's (unless by_length); most shares
  bool causal, bf16, partial;                       // partial: part_o and part_ml are the result
  bool split, by_length;                            // items of the last round are halved; tiles per share follow from the lengths (prompt.cu)
  float scale_log2;                                 // scale * log2(e)
  void* out;                                        // [total_q][nh_q][128]
  float* lse;                                       // [nh_q][total_q]
  float* part_o;                                    // [shares][total_q * nh_q][128], not yet normalised
  float2* part_ml;                                  // [shares][total_q * nh_q] (maximum, sum), in powers of two
  int* share_size;                                  // by_length: what the kernel has chosen
};

struct PromptMaps {   // the tensors as (channel, head, token), for copies by tiles
  CUtensorMap q, k, v, pk, pv;
};

// Attention of p's queries (a token each, no sequences) to its prefix alone, in parts to be joined; how many.
int prefix_parts(const hqkv_prompt_t* p);
int prefix_partial(const hqkv_prompt_t* p, float* part_o, float2* part_ml, cudaStream_t st);

}  // namespace hqkv
