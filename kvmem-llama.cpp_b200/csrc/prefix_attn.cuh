// Attention of a batch of sequences over a shared prefix and their own tails.
#pragma once

#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

#include "qkv.cuh"

namespace kvmret {

// The keys of one kind: a list of pages and how many tokens of it count.
struct KeyList {
    PageView pages;
    const int32_t *table;    // page ids; null: 0, 1, 2, ...
    const uint32_t *ntok;    // tokens held by each listed page; null: full
    const int32_t *len;      // tokens (device; with ntok: of those that the pages hold); null: max_len
    uint32_t max_len;        // bound on the tokens (0: no such keys)
    uint32_t n_list;         // pages of one list
};

struct PrefixAttn {
    const uint16_t *q;       // f16 rows of n_head * D elements
    uint64_t q_stride;
    uint16_t *out;           // f16 [n_q][n_head][D]
    float *lse;              // [n_q][n_head] or null
    uint32_t n_q, n_head, n_head_kv, d_head;
    float scale;
    KeyList prefix;          // one list, for every row
    KeyList tail;            // n_seq lists; len: [n_seq]
    uint32_t n_seq;
    const int32_t *q_start;  // [n_seq + 1] first row of each sequence
};
size_t prefix_attn_ws_bytes(uint32_t n_q, uint32_t n_head, uint32_t n_head_kv, uint32_t d_head,
                            uint32_t n_seq);
cudaError_t launch_prefix_attn(const PrefixAttn &a, void *ws, cudaStream_t st);

}  // namespace kvmret
