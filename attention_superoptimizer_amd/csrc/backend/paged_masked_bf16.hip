// Attention over a paged key-value cache of trees and of windows beside a sequence's first keys: the kernels of bf16 values
// (paged_attention.h).
#include "paged_attention.h"

int mi355::paged::launch_masked_bf16(MaskedParams const &P, int kv_heads, bool passing, bool tree) {
  return tree ? launch_head<__bf16, kTree>(P, kv_heads, passing) : launch_head<__bf16, kFirstKeys>(P, kv_heads, passing);
}
