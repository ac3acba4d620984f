// Attention over a paged key-value cache: its kernels of bf16 values.
#include "paged_attention.h"

namespace mi355 {
int paged::launch_bf16(PagedParams const &P, int kv_heads, bool passing) { return launch_head<__bf16>(P, kv_heads, passing); }
}  // namespace mi355
