// Argument checks shared by the entry points on paged caches.
#pragma once

#include "kvmret.h"
#include "prefix_attn.cuh"

namespace kvmret {

// Records a message for kvmret_last_error() and returns the code (context.cpp).
int set_error(int code, const char *msg);

// Checks a page description and resolves it (strides of 0, row bytes).
// Returns KVMRET_OK or the recorded error.
int resolve_pages(const kvmret_pages *p, const char *what, PageView *out);

// kvmret_prefix_attn with the prefix given as a resolved key list (max_len 0:
// none): checks the rest, launches.
int prefix_attn_call(const KeyList &prefix, const kvmret_pages *tail, const kvmret_attn *a,
                     void *ws, size_t ws_bytes, cudaStream_t st);

}  // namespace kvmret
