// Eviction from KV caches by accumulated attention weight (cache_evict.cu).
#pragma once

#include "launch.h"

namespace dl {

struct EvictArgs {
  int caches, kv_heads, width, capacity, out_capacity;
  int budget;  // <= capacity
  int first, recent;
  bool in_place;
  const bf16 *key, *value;
  size_t row_stride, cache_stride;
  const float* weights;
  const int* positions;
  const long long* lengths;
  bf16 *key_out, *value_out;
  size_t out_row_stride, out_cache_stride;
  float* weights_out;
  int* positions_out;
  long long* lengths_out;
};

size_t cache_evict_workspace_bytes(int caches, int kv_heads, int budget);
int cache_evict_most_slots();  // of one (cache, KV head)
cudaError_t launch_cache_evict(const EvictArgs& a, void* workspace, int sms, cudaStream_t stream);

}  // namespace dl
