// Attention of a sequence's new tokens over a paged key-value cache.
//
// o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q . k_j, over the keys a row sees, in one pass with the
// running maximum m: when it grows, what has been summed is scaled down.
#include "common.h"

#include <climits>
#include <cmath>

namespace mi355 {

int check_paged_cache(mi355_paged_cache const &c) {
  if (c.k == nullptr || c.v == nullptr || c.k == c.v) {
    return fail(MI355_ERR_INVALID, "paged cache: keys and values are two tensors");
  }
  if (c.pages < 1 || c.page_size < 1 || c.kv_heads < 1 || c.head_dim < 1 || (long long)c.pages * c.page_size > INT_MAX ||
      c.page_stride < 0 || c.token_stride < 0 || c.head_stride < 0) {
    return fail(MI355_ERR_INVALID, "paged cache: %d pages of %d, %d heads of %d", c.pages, c.page_size, c.kv_heads, c.head_dim);
  }
  if (c.type != MI355_TYPE_F16 && c.type != MI355_TYPE_BF16) {
    return fail(MI355_ERR_UNSUPPORTED, "paged cache: type %d", c.type);
  }
  return MI355_OK;
}

namespace {

struct PagedParams {
  void const *q, *k, *v;
  void *out;
  long long q_stride, out_stride, page_stride, token_stride, head_stride;
  int const *table, *lengths;
  int pages, page_size, kv_heads, head_dim, table_width, sequences, new_tokens, group, window;
  float scale;
};

// One wavefront per row (new token, query head); 64 keys at a time, a key a lane for the scores, 64 columns at a time
// for the values.
template <class T>
__global__ __launch_bounds__(64) void paged_attention_kernel(PagedParams const P) {
  __shared__ float q[MI355_MAX_PAGED_HEAD_DIM], weight[64];
  __shared__ long long place[64];
  int const row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, kv = head / P.group;
  int const sequence = row / P.new_tokens, t = row % P.new_tokens, D = P.head_dim;
  T const *const query = static_cast<T const *>(P.q) + row * P.q_stride + (long long)head * D;
  for (int d = lane; d < D; d += 64) {
    q[d] = static_cast<float>(query[d]) * P.scale;
  }
  __syncthreads();
  int const most = P.table_width * P.page_size, told = P.lengths[sequence], length = told < 0 ? 0 : (told < most ? told : most);
  int const end = length - (P.new_tokens - 1 - t), begin = P.window != 0 && end > P.window ? end - P.window : 0;
  int const *const table = P.table + (long long)sequence * P.table_width;
  float m = -INFINITY, sum = 0.0f, acc[MI355_MAX_PAGED_HEAD_DIM / 64] = {};
  for (int base = begin; base < end; base += 64) {
    int const key = base + lane;
    int const page = key < end ? table[key / P.page_size] : -1;
    bool const seen = page >= 0 && page < P.pages;
    long long const at = seen ? page * P.page_stride + (long long)(key % P.page_size) * P.token_stride + kv * P.head_stride : 0;
    float s = -INFINITY;
    if (seen) {
      s = 0.0f;
      for (int d = 0; d < D; d++) {
        s += q[d] * static_cast<float>(static_cast<T const *>(P.k)[at + d]);
      }
    }
    float top = s;
    for (int off = 32; off > 0; off >>= 1) {
      top = fmaxf(top, __shfl_xor(top, off, 64));
    }
    float const higher = fmaxf(m, top);
    if (__all(!seen)) {
      continue;
    }
    // (no score above minus infinity yet: nothing to scale, no weight)
    float const scaled = m == -INFINITY ? 0.0f : expf(m - higher), w = seen && s != -INFINITY ? expf(s - higher) : 0.0f;
    m = higher;
    weight[lane] = w;
    place[lane] = seen ? at : -1;
    float total = w;
    for (int off = 32; off > 0; off >>= 1) {
      total += __shfl_xor(total, off, 64);
    }
    sum = sum * scaled + total;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI355_MAX_PAGED_HEAD_DIM / 64; i++) {
      int const d = 64 * i + lane;
      if (d < D) {
        float a = acc[i] * scaled;
        for (int j = 0; j < 64; j++) {
          if (place[j] >= 0) {
            a += weight[j] * static_cast<float>(static_cast<T const *>(P.v)[place[j] + d]);
          }
        }
        acc[i] = a;
      }
    }
    __syncthreads();
  }
  T *const out = static_cast<T *>(P.out) + row * P.out_stride + (long long)head * D;
#pragma unroll
  for (int i = 0; i < MI355_MAX_PAGED_HEAD_DIM / 64; i++) {
    int const d = 64 * i + lane;
    if (d < D) {
      out[d] = static_cast<T>(sum == 0.0f ? 0.0f : acc[i] / sum);
    }
  }
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355_paged_attention(void const *q, long long q_stride, void *out, long long out_stride,
                                     mi355_paged_cache const *cache, int const *table, int table_width, int const *lengths,
                                     int sequences, int new_tokens, int q_heads, float scale, int window) {
  MI355_REQUIRE_INIT();
  if (cache == nullptr) {
    return fail(MI355_ERR_INVALID, "mi355_paged_attention: null cache");
  }
  mi355_paged_cache const &c = *cache;
  if (int rc = check_paged_cache(c)) {
    return rc;
  }
  if (sequences < 0 || new_tokens < 1 || q_heads < 1 || q_heads % c.kv_heads != 0 || table_width < 1 || window < 0 ||
      !std::isfinite(scale) || q_stride < 0 || out_stride < 0) {
    return fail(MI355_ERR_INVALID, "mi355_paged_attention: %d sequences of %d new tokens, %d heads over %d, table of %d, window %d",
                sequences, new_tokens, q_heads, c.kv_heads, table_width, window);
  }
  if (c.head_dim % 8 != 0 || c.head_dim > MI355_MAX_PAGED_HEAD_DIM || (long long)table_width * c.page_size > INT_MAX - 1024 ||
      (long long)sequences * new_tokens > INT_MAX || q_heads > 65535) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_paged_attention: heads of %d, a table of %d pages of %d, %d x %d tokens, %d heads",
                c.head_dim, table_width, c.page_size, sequences, new_tokens, q_heads);
  }
  if (sequences == 0) {
    return MI355_OK;
  }
  if (q == nullptr || out == nullptr || table == nullptr || lengths == nullptr) {
    return fail(MI355_ERR_INVALID, "mi355_paged_attention: null pointer");
  }
  uintptr_t const bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(c.k) |
                         reinterpret_cast<uintptr_t>(c.v);
  if (bits % 16 != 0 || (q_stride | out_stride | c.page_stride | c.token_stride | c.head_stride) % 8 != 0) {
    return fail(MI355_ERR_INVALID, "mi355_paged_attention: tensors begin, and their strides step, 16 bytes at a time");
  }
  PagedParams P;
  P.q = q;
  P.k = c.k;
  P.v = c.v;
  P.out = out;
  P.q_stride = q_stride;
  P.out_stride = out_stride;
  P.page_stride = c.page_stride;
  P.token_stride = c.token_stride;
  P.head_stride = c.head_stride;
  P.table = table;
  P.lengths = lengths;
  P.pages = c.pages;
  P.page_size = c.page_size;
  P.kv_heads = c.kv_heads;
  P.head_dim = c.head_dim;
  P.table_width = table_width;
  P.sequences = sequences;
  P.new_tokens = new_tokens;
  P.group = q_heads / c.kv_heads;
  P.window = window;
  P.scale = scale;
  auto *fn = c.type == MI355_TYPE_F16 ? paged_attention_kernel<_Float16> : paged_attention_kernel<__bf16>;
  MI355_HIP(launch_kernel(fn, dim3((unsigned)(sequences * new_tokens), (unsigned)q_heads), dim3(64), 0, state().stream(), P));
  return MI355_OK;
}
