// Attention over a paged key-value cache: its entry point, and its kernels of fp16 values (paged_attention.h).
#include "paged_attention.h"

namespace mi355 {

int paged::launch_f16(PagedParams const &P, int kv_heads, bool passing) { return launch_head<_Float16>(P, kv_heads, passing); }

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
}  // namespace mi355

using namespace mi355;
using namespace mi355::paged;

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
  long long const keys = (long long)table_width * c.page_size;
  if (c.head_dim % 8 != 0 || c.head_dim > MI355_MAX_PAGED_HEAD_DIM || keys > 1 << 30 || (long long)sequences * new_tokens > INT_MAX ||
      (long long)new_tokens * q_heads > 1 << 29 || (long long)q_heads * c.head_dim > INT_MAX) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_paged_attention: heads of %d, a table of %d pages of %d, %d x %d tokens, %d heads",
                c.head_dim, table_width, c.page_size, sequences, new_tokens, q_heads);
  }
  if ((long long)sequences * new_tokens > 1 && out_stride < (long long)q_heads * c.head_dim) {
    return fail(MI355_ERR_INVALID, "mi355_paged_attention: results of %d heads of %d lie %lld apart", q_heads, c.head_dim, out_stride);
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
  auto steps = [](long long stride, int n) { return stride / 8 > UINT32_MAX ? UINT32_MAX : (long long)(n - 1) * (stride / 8); };
  if (steps(c.page_stride, c.pages) > UINT32_MAX || steps(c.token_stride, c.page_size) > UINT32_MAX || steps(c.head_stride, c.kv_heads) > UINT32_MAX ||
      steps(c.page_stride, c.pages) + steps(c.token_stride, c.page_size) + steps(c.head_stride, c.kv_heads) + c.head_dim / 8 >= UINT32_MAX) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_paged_attention: keys or values of more than 64 GB");
  }
  PagedParams P{};
  P.q = q;
  P.k = c.k;
  P.v = c.v;
  P.out = out;
  P.q_stride = q_stride;
  P.out_stride = out_stride;
  P.page_step = (uint32_t)(c.page_stride / 8);
  P.token_step = (uint32_t)(c.token_stride / 8);
  P.head_step = (uint32_t)(c.head_stride / 8);
  P.table = table;
  P.lengths = lengths;
  P.parts = static_cast<float *>(state().scratch());
  P.tickets = state().queue_join_tickets();
  P.pages = c.pages;
  P.page_size = c.page_size;
  P.head_dim = c.head_dim;
  P.table_width = table_width;
  P.new_tokens = new_tokens;
  P.group = q_heads / c.kv_heads;
  P.window = window < keys ? window : 0;
  P.page_magic = magic_of(c.page_size);
  P.group_magic = magic_of(P.group);
  P.q_keep = scale == 0.0f ? 0 : ~0u;
  P.q_flip = scale < 0.0f ? 0x80008000u : 0;
  P.scale = scale == 0.0f ? 1.0f : fabsf(scale) * 1.44269504088896341f;
  // Loads that are not to be kept in the caches, from three quarters of the 256 MB on that the last-level cache holds: measured
  // (us, kept and not) 106 and 95 of 539 MB in 64 sequences, 49.5 and 45.8 of 201 MB in 24, 53.6 and 47.6 of 255 MB in 9; against it
  // 31.6 and 32.4 of 150 MB in 16, 28.2 and 29.3 of 136 MB in 14.
  long long const slots = (long long)sequences * keys < (long long)c.pages * c.page_size ? (long long)sequences * keys : (long long)c.pages * c.page_size;
  bool const passing = 4 * slots * c.kv_heads * c.head_dim > 192LL << 20;
  // units are counted in 32 bits: a batch with more of them goes in slices of sequences
  long long const rows = (long long)new_tokens * P.group;
  if (too_many_units(c.kv_heads, rows, keys)) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_paged_attention: %d new tokens of %d heads over %lld keys", new_tokens, q_heads, keys);
  }
  long long const slice = sequences_at_once(c.kv_heads, rows, keys);
  for (long long at = 0; at < sequences; at += slice) {
    P.sequences = (int)(sequences - at < slice ? sequences - at : slice);
    P.q = static_cast<char const *>(q) + 2 * at * new_tokens * q_stride;
    P.out = static_cast<char *>(out) + 2 * at * new_tokens * out_stride;
    P.table = table + at * table_width;
    P.lengths = lengths + at;
    if (int rc = c.type == MI355_TYPE_F16 ? launch_f16(P, c.kv_heads, passing) : launch_bf16(P, c.kv_heads, passing)) {
      return rc;
    }
  }
  return MI355_OK;
}
