// kvcache.cuh -- kernel-side view of the paged HiF4 key/value cache.
#pragma once
#include "common.cuh"

namespace hif4x {

struct CacheArgs {
  uint8_t *codes[2];     // K, V: (pages, heads, page_size, dh/2)
  uint32_t *meta[2];     // (pages, heads, page_size, dh/64)
  int64_t num_pages;
  int heads, page_size, page_shift, nb;   // nb = dh / 64
  const int *cu_new, *kv_len, *pages;
  int B, most;           // sequences; entries of a row of `pages` that count
  int64_t ld_pages, rows;
  int *status;           // [0] of the bounded waits, [1] of the page tables
};

// csrc/kvcache.cu: checks a cache and batch description and fills the arguments
int cache_args(const hif4x_kv_cache *kv, const hif4x_kv_batch *b, int64_t rows, CacheArgs *a);

}  // namespace hif4x
