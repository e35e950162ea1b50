// Argument checks shared by the entry points on paged caches.
#pragma once

#include "kvmret.h"
#include "qkv.cuh"

namespace kvmret {

// Records a message for kvmret_last_error() and returns the code (context.cpp).
int set_error(int code, const char *msg);

// Checks a page description and resolves it (strides of 0, row bytes).
// Returns KVMRET_OK or the recorded error.
int resolve_pages(const kvmret_pages *p, const char *what, PageView *out);

}  // namespace kvmret
