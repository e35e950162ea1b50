// Per-head norms with the position rotation, and the append of keys and
// values to a paged cache. Launches are asynchronous on the given stream.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

#include "kernels.cuh"

namespace kvmret {

// Element types of the activations (ggml type ids).
enum { kTypeF32 = 0, kTypeBF16 = 30 };

struct QkNormRope {
    const void *q, *k;           // rows of `type`: head h of token t at t * stride + h * D
    uint64_t q_stride, k_stride; // elements between tokens
    const float *q_weight, *k_weight;  // [D] or null (ones)
    const int32_t *pos;          // [n_tok]
    uint16_t *q_rot, *k_rot, *q_raw, *k_raw;  // f16 [n_tok][heads][D], null: not wanted
    uint32_t n_tok, n_head, n_head_kv, d_head;
    int32_t type;                // kTypeF32, KVMRET_TYPE_F16 or kTypeBF16
    float eps;
    uint32_t fwht_n;             // 0 or d_head: Hadamard transform of the rotated rows
    Theta theta;
};
cudaError_t launch_qk_norm_rope(const QkNormRope &a, cudaStream_t st);

// A paged cache: token `off` of page p has its K row at k + p * k_page +
// off * k_row, its V row likewise.
struct PageView {
    uint8_t *k, *v;
    uint64_t k_page, v_page, k_row, v_row;
    uint32_t n_pages, page_tokens, n_head_kv, d_head;
    int32_t k_type, v_type;
};

struct PagedAppend {
    PageView pages;
    const uint16_t *k, *v;       // f16 rows of Hkv * D elements
    uint64_t k_stride, v_stride; // elements between tokens
    const int32_t *cells;        // [n_tok]: page * page_tokens + offset; others are skipped
    const int32_t *pos;          // [n_tok], null: K is stored unrotated
    uint32_t n_tok;
    uint32_t fwht_n;
    Theta theta;
};
cudaError_t launch_paged_append(const PagedAppend &a, cudaStream_t st);

}  // namespace kvmret
