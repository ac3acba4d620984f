// Attention of trees and within windows over a paged key-value cache: entry points, and the kernels of fp16 values
// (attention_blocks.h).
#include "attention_blocks.h"
#include "slices.h"

namespace mi355 {

int blocks::launch_f16(BlockParams const &P, bool tree) { return tree ? launch_head<_Float16, true>(P) : launch_head<_Float16, false>(P); }

namespace {

using namespace blocks;

// What both entry points take; `name` is the caller's.  P is filled but for what masks are made of.
int fill(BlockParams &P, char const *name, void const *q, long long q_stride, void *out, long long out_stride, mi355_paged_cache const &c,
         int const *table, int table_width, int const *lengths, int sequences, long long tokens, bool ragged, int q_heads, float scale) {
  if (sequences < 0 || q_heads < 1 || q_heads % c.kv_heads != 0 || table_width < 1 || !std::isfinite(scale) || q_stride < 0 || out_stride < 0) {
    return fail(MI355_ERR_INVALID, "%s: %d sequences, %d heads over %d, table of %d", name, sequences, q_heads, c.kv_heads, table_width);
  }
  long long const keys = (long long)table_width * c.page_size;
  if (c.head_dim % 8 != 0 || c.head_dim > MI355_MAX_PAGED_HEAD_DIM || keys > 1 << 30 || tokens > INT_MAX ||
      (long long)q_heads * c.head_dim > INT_MAX || !fit(tokens, q_heads / c.kv_heads, c.kv_heads, sequences, ragged)) {
    return fail(MI355_ERR_UNSUPPORTED, "%s: heads of %d, a table of %d pages of %d, %lld tokens, %d heads", name, c.head_dim, table_width,
                c.page_size, tokens, q_heads);
  }
  if (tokens > 1 && out_stride < (long long)q_heads * c.head_dim) {
    return fail(MI355_ERR_INVALID, "%s: results of %d heads of %d lie %lld apart", name, q_heads, c.head_dim, out_stride);
  }
  if (tokens == 0 || sequences == 0) {
    return MI355_OK;
  }
  if (q == nullptr || out == nullptr || table == nullptr || lengths == nullptr) {
    return fail(MI355_ERR_INVALID, "%s: null pointer", name);
  }
  uintptr_t const bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(c.k) |
                         reinterpret_cast<uintptr_t>(c.v);
  if (bits % 16 != 0 || (q_stride | out_stride | c.page_stride | c.token_stride | c.head_stride) % 8 != 0) {
    return fail(MI355_ERR_INVALID, "%s: tensors begin, and their strides step, 16 bytes at a time", name);
  }
  auto steps = [](long long stride, int n) { return stride / 8 > UINT32_MAX ? UINT32_MAX : (long long)(n - 1) * (stride / 8); };
  if (steps(c.page_stride, c.pages) > UINT32_MAX || steps(c.token_stride, c.page_size) > UINT32_MAX || steps(c.head_stride, c.kv_heads) > UINT32_MAX ||
      steps(c.page_stride, c.pages) + steps(c.token_stride, c.page_size) + steps(c.head_stride, c.kv_heads) + c.head_dim / 8 >= UINT32_MAX) {
    return fail(MI355_ERR_UNSUPPORTED, "%s: keys or values of more than 64 GB", name);
  }
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
  P.pages = c.pages;
  P.page_size = c.page_size;
  P.head_dim = c.head_dim;
  P.table_width = table_width;
  P.sequences = sequences;
  P.tokens = (int)tokens;
  P.group = q_heads / c.kv_heads;
  P.kv_heads = c.kv_heads;
  P.page_magic = paged::magic_of(c.page_size);
  P.group_magic = paged::magic_of(P.group);
  P.q_keep = scale == 0.0f ? 0 : ~0u;
  P.q_flip = scale < 0.0f ? 0x80008000u : 0;
  P.scale = scale == 0.0f ? 1.0f : fminf(fabsf(scale) * 1.44269504088896341f, FLT_MAX);  // (a score of zero stays zero)
  return MI355_OK;
}

// Few rows of a key-value head, as many in every sequence: a head's keys are dealt over workgroups, a wavefront has 32 of them at a time to
// itself (paged_attention.h), and reading the cache is what counts.  Measured (us, that and blocks; heads of 128 unless said): 11.4 and 16.0 of 1
// sequence x 8 heads within a window of 4096, 4 rows, 85 and 106 of 64 x 8 within 2048, 4 rows, 10.4 and 12.9 of 1 x 8 x 1000 keys, 8 rows, 19.9 and 25.2
// of 8 x 8 within 2048, 16 rows, 51 and 68 of 16 x 8 heads of 256 within 2048, 16 rows; against it 41 and 39 of 32 x 8 heads of 64 x up to 4096, 16
// rows, 24.1 and 21.4 of 5 x 3 heads of 256 x up to 3001, 15 rows, and with 32 rows 56 and 40 of the same heads of 64, 86 and 64 of 32 x 8 x up to 4096,
// 16.4 and 12.4 of 1 x 8 x 1000.
bool few_rows(BlockParams const &P) {
  long long const rows = (long long)P.new_tokens * P.group;
  return P.starts == nullptr && rows <= 16 && !paged::too_many_units(P.kv_heads, rows, (long long)P.table_width * P.page_size);
}

int launch_few(BlockParams const &B, int type, bool tree) {
  paged::MaskedParams P{};
  P.k = B.k;
  P.v = B.v;
  P.q_stride = B.q_stride;
  P.out_stride = B.out_stride;
  P.page_step = B.page_step;
  P.token_step = B.token_step;
  P.head_step = B.head_step;
  P.parts = static_cast<float *>(state().scratch());
  P.tickets = state().queue_join_tickets();
  P.pages = B.pages;
  P.page_size = B.page_size;
  P.head_dim = B.head_dim;
  P.table_width = B.table_width;
  P.new_tokens = B.new_tokens;
  P.group = B.group;
  P.window = B.window;
  P.page_magic = B.page_magic;
  P.group_magic = B.group_magic;
  P.q_keep = B.q_keep;
  P.q_flip = B.q_flip;
  P.scale = B.scale;
  P.sinks = B.sinks;
  long long const keys = (long long)B.table_width * B.page_size, rows = (long long)B.new_tokens * B.group;
  P.most_keys = (int)paged::keys_seen(keys, B.window, B.sinks, B.new_tokens);
  // loads that pass the caches: as in mi355_paged_attention
  long long const visible = (long long)B.sequences * P.most_keys, all = (long long)B.pages * B.page_size;
  bool const passing = 4 * (visible < all ? visible : all) * B.kv_heads * B.head_dim > 192LL << 20;
  long long const slice = paged::masked_at_once(B.kv_heads, rows, P.most_keys);
  return in_slices(B.sequences, slice, [&](long long at, long long count) -> int {
    P.sequences = (int)count;
    P.q = static_cast<char const *>(B.q) + 2 * at * B.new_tokens * B.q_stride;
    P.out = static_cast<char *>(B.out) + 2 * at * B.new_tokens * B.out_stride;
    P.table = B.table + at * B.table_width;
    P.lengths = B.lengths + at;
    P.parents = tree ? B.parents + at * B.new_tokens : nullptr;
    return type == MI355_TYPE_F16 ? paged::launch_masked_f16(P, B.kv_heads, passing, tree) : paged::launch_masked_bf16(P, B.kv_heads, passing, tree);
  });
}

int launch(BlockParams &P, int type, bool tree) {
  if (few_rows(P)) {
    return launch_few(P, type, tree);
  }
  auto run = [&](BlockParams const &Q) { return type == MI355_TYPE_F16 ? launch_f16(Q, tree) : launch_bf16(Q, tree); };
  if (P.starts != nullptr) {
    return run(P);
  }
  long long const slice = sequences_at_once((long long)P.new_tokens * P.group, P.kv_heads);
  return in_slices(P.sequences, slice, [&](long long at, long long count) -> int {
    BlockParams Q = P;
    Q.sequences = (int)count;
    Q.tokens = (int)(count * P.new_tokens);
    Q.q = static_cast<char const *>(P.q) + 2 * at * P.new_tokens * P.q_stride;
    Q.out = static_cast<char *>(P.out) + 2 * at * P.new_tokens * P.out_stride;
    Q.table = P.table + at * P.table_width;
    Q.lengths = P.lengths + at;
    Q.parents = tree ? P.parents + at * P.new_tokens : nullptr;
    return run(Q);
  });
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355_tree_attention(void const *q, long long q_stride, void *out, long long out_stride, mi355_paged_cache const *cache,
                                    int const *table, int table_width, int const *lengths, int const *parents, int sequences, int nodes,
                                    int q_heads, float scale) {
  MI355_REQUIRE_INIT();
  if (cache == nullptr) {
    return fail(MI355_ERR_INVALID, "mi355_tree_attention: null cache");
  }
  if (int rc = check_paged_cache(*cache)) {
    return rc;
  }
  if (nodes < 1 || nodes > MI355_MAX_TREE_NODES) {
    return fail(nodes < 1 ? MI355_ERR_INVALID : MI355_ERR_UNSUPPORTED, "mi355_tree_attention: trees of %d nodes", nodes);
  }
  blocks::BlockParams P{};
  if (int rc = fill(P, "mi355_tree_attention", q, q_stride, out, out_stride, *cache, table, table_width, lengths, sequences,
                    (long long)sequences * nodes, false, q_heads, scale)) {
    return rc;
  }
  if (sequences == 0) {
    return MI355_OK;
  }
  if (parents == nullptr) {
    return fail(MI355_ERR_INVALID, "mi355_tree_attention: null pointer");
  }
  P.parents = parents;
  P.new_tokens = nodes;
  return launch(P, cache->type, true);
}

extern "C" int mi355_window_attention(void const *q, long long q_stride, void *out, long long out_stride, mi355_paged_cache const *cache,
                                      int const *table, int table_width, int const *lengths, int const *starts, int sequences, int tokens,
                                      int q_heads, float scale, int window, int sinks) {
  MI355_REQUIRE_INIT();
  if (cache == nullptr) {
    return fail(MI355_ERR_INVALID, "mi355_window_attention: null cache");
  }
  if (int rc = check_paged_cache(*cache)) {
    return rc;
  }
  if (tokens < 0 || window < 0 || sinks < 0 || (starts == nullptr && (sequences > 0 ? tokens % sequences != 0 : tokens != 0))) {
    return fail(MI355_ERR_INVALID, "mi355_window_attention: %d tokens of %d sequences, window %d, %d kept", tokens, sequences, window, sinks);
  }
  blocks::BlockParams P{};
  if (int rc = fill(P, "mi355_window_attention", q, q_stride, out, out_stride, *cache, table, table_width, lengths, sequences, tokens,
                    starts != nullptr, q_heads, scale)) {
    return rc;
  }
  if (sequences == 0 || tokens == 0) {
    return MI355_OK;
  }
  long long const keys = (long long)table_width * cache->page_size;
  P.starts = starts;
  P.new_tokens = starts == nullptr ? tokens / sequences : 0;
  P.window = window < keys ? window : 0;
  P.sinks = P.window == 0 ? 0 : (sinks < keys ? sinks : (int)keys);
  return launch(P, cache->type, false);
}
