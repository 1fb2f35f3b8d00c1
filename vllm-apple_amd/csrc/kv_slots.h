// Where a token's K/V row lies in the paged cache: the resolvers of the KV
// write and of the quantised write and read.  Each returns false for a token
// without a slot, which the kernels skip.
#pragma once

#include "common.h"

namespace vaa {

// slot_mapping (kv_write.py:130-146): block = slot / bs, offset = slot % bs.
template <typename IdxT>
struct SlotResolver {
  const IdxT* slots;
  int block_size;
  int64_t capacity;  // num_blocks * block_size
  __device__ bool operator()(int t, int64_t& block, int64_t& off) const {
    int64_t s = static_cast<int64_t>(slots[t]);
    if (s < 0 || s >= capacity) return false;
    block = s / block_size;
    off = s % block_size;
    return true;
  }
};

// Decode position (paged_attention_fused.metal:73-86, kv_write.py:86-99).
struct DecodeResolver {
  const int32_t* block_table;
  const int32_t* seq_lens;
  int max_blocks_per_seq;
  int block_size;
  int64_t num_blocks;
  __device__ bool operator()(int s, int64_t& block, int64_t& off) const {
    int L = seq_lens[s];
    if (L <= 0) return false;
    int pos = L - 1;
    int bi = pos / block_size;
    if (bi >= max_blocks_per_seq) return false;
    int phys = block_table[static_cast<int64_t>(s) * max_blocks_per_seq + bi];
    if (phys < 0 || phys >= num_blocks) return false;
    block = phys;
    off = pos % block_size;
    return true;
  }
};

}  // namespace vaa
