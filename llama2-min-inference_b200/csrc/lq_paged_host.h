// Host checks shared by the paged-cache entry points (C++ only).
#pragma once
#include "lq_host.h"

namespace lq {

// arguments that kv_append and paged_attention have in common
int check_paged(const PagedKV* c, const KVBatch* b, int n_heads, int type, const char* fn);

}  // namespace lq
