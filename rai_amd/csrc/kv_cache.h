// A key/value cache in pages of 8-bit codes (kv_cache.hip writes it, kv_attention.hip reads it):
//   k [pages][heads][page][features], v [pages][heads][features][page], one scale for each page and head of each.
// Values lie transposed so that sixteen tokens of a feature are 16 bytes: the fragments of the attention's second product
// then come from memory as they lie, like the keys' of its first.
#pragma once
#include "common.h"

namespace rai {

constexpr int kKvMaxFeatures = 256;

struct KvCacheView {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int64_t pages;
  int heads, page, page_shift, features;   // page = 1 << page_shift tokens
  int format;
};
// Checks the five arguments every entry point of the cache takes.
int kv_cache_view(const char *what, int32_t format, const rai_hip_tensor *k, const rai_hip_tensor *v, const rai_hip_tensor *k_scale,
                  const rai_hip_tensor *v_scale, KvCacheView *out);

// Whether the bytes that two tensors span (their strides' extremes) have one in common.
bool overlap(const rai_hip_tensor *a, const rai_hip_tensor *b);

}  // namespace rai
