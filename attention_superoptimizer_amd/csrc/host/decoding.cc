// Operators of a decoding step (include/mirage/kernel/decoding.h): what they take, their results' tensors, and the
// calls of the C ABI that run them.
#include "mi355_abi.h"
#include "mi355_kernels/paged_units.h"
#include "mirage/kernel/device_memory_manager.h"
#include "mirage/kernel/graph.h"
#include "mirage/utils/hip_types.h"
#include "mirage/utils/json_utils.h"

#include <climits>
#include <cmath>
#include <initializer_list>

namespace mirage {
namespace kernel {

using namespace mirage::type;

#define MI355_CALL(expr) MIRAGE_CHECK((expr) == MI355_OK, mi355_last_error())

char const *without_kernel(KNOperator const &op);  // (kernel_device.cc)

namespace {

bool row_major(DTensor const &t) { return t.layout == mirage::layout::DmemRowMajor; }

bool has_dims(DTensor const &t, std::initializer_list<int> dims) {
  if (t.num_dims != (int)dims.size()) {
    return false;
  }
  int i = 0;
  for (int d : dims) {
    if (t.dim[i++] != d) {
      return false;
    }
  }
  return true;
}

bool positive(DTensor const &t) {
  for (int i = 0; i < t.num_dims; i++) {
    if (t.dim[i] <= 0) {
      return false;
    }
  }
  return t.num_dims > 0;
}

bool half_type(DTensor const &t) { return t.data_type == DT_FLOAT16 || t.data_type == DT_BFLOAT16; }

// Whether results of these element counts, each with its fingerprint buffer, fit the arena.
bool room_for(std::initializer_list<size_t> data_bytes, std::initializer_list<size_t> fingerprint_bytes) {
  size_t need = 0;
  for (auto const &list : {data_bytes, fingerprint_bytes}) {
    for (size_t b : list) {
      need += (b + 15) / 16 * 16;
    }
  }
  return DeviceMemoryManager::get_instance()->has_room(need);
}
bool room_for(DTensor const &t) { return room_for({t.data_size()}, {t.fingerprint_size()}); }

void adopt(KNOperator *op, DTensor t) {
  t.owner_op = op;
  t.owner_ts_idx = (int)op->output_tensors.size();
  t.guid = DTensor::next_guid++;
  DeviceMemoryManager::get_instance()->allocate(t);
  op->output_tensors.push_back(t);
}

DTensor tensor_of(std::initializer_list<int> dims, DataType type) {
  DTensor t;
  for (int d : dims) {
    t.dim[t.num_dims++] = d;
  }
  t.layout = mirage::layout::DmemRowMajor;
  t.data_type = type;
  return t;
}

struct CacheShape {
  int pages, page_size, kv_heads, head_dim;
  CacheShape(DTensor const &t, bool heads_first)
      : pages(t.dim[0]), page_size(t.dim[heads_first ? 2 : 1]), kv_heads(t.dim[heads_first ? 1 : 2]), head_dim(t.dim[3]) {}
};

// two caches of one shape and type, and not the same tensor
bool caches_ok(DTensor const &k, DTensor const &v, bool heads_first) {
  if (k.num_dims != 4 || !positive(k) || !half_type(k) || v.data_type != k.data_type || !row_major(k) || !row_major(v) ||
      !has_dims(v, {k.dim[0], k.dim[1], k.dim[2], k.dim[3]}) || k.data_ptr == v.data_ptr) {
    return false;
  }
  CacheShape const c(k, heads_first);
  return (long long)c.pages * c.page_size <= INT_MAX;
}

mi355_paged_cache cache_of(DTensor const &k, DTensor const &v, bool heads_first) {
  CacheShape const c(k, heads_first);
  mi355_paged_cache p;
  p.k = k.data_ptr;
  p.v = v.data_ptr;
  p.pages = c.pages;
  p.page_size = c.page_size;
  p.kv_heads = c.kv_heads;
  p.head_dim = c.head_dim;
  p.page_stride = (long long)c.page_size * c.kv_heads * c.head_dim;
  p.token_stride = (long long)c.head_dim * (heads_first ? 1 : c.kv_heads);
  p.head_stride = (long long)c.head_dim * (heads_first ? c.page_size : 1);
  p.type = k.data_type;
  return p;
}

// heads of `head_dim` elements in a row of [tokens, heads, head_dim] or [tokens, heads * head_dim]; 0: neither
int heads_in(DTensor const &t, int head_dim) {
  if (t.num_dims == 3 && t.dim[2] == head_dim) {
    return t.dim[1];
  }
  return t.num_dims == 2 && t.dim[1] % head_dim == 0 ? t.dim[1] / head_dim : 0;
}

bool angles_ok(DTensor const &positions, DTensor const &angles, int tokens, int head_dim) {
  return positive(positions) && positive(angles) && has_dims(positions, {tokens}) && positions.data_type == DT_INT32 && row_major(positions) && angles.num_dims == 2 &&
         angles.dim[0] == 2 && angles.dim[1] <= head_dim / 2 && angles.dim[1] <= MI355_MAX_ROTARY_PAIRS && angles.data_type == DT_DOUBLE && row_major(angles);
}

bool rotary_ok(DTensor const &x, DTensor const &positions, DTensor const &angles) {
  return x.num_dims == 3 && positive(x) && half_type(x) && row_major(x) && (long long)x.dim[1] * x.dim[2] <= 1 << 30 &&
         angles_ok(positions, angles, x.dim[0], x.dim[2]);
}

// queries' heads of the projection; 0: infeasible
int append_q_heads(DTensor const &qkv, DTensor const &positions, DTensor const &angles, DTensor const &slots, DTensor const &k,
                   DTensor const &v, bool heads_first) {
  if (!caches_ok(k, v, heads_first) || qkv.data_type != k.data_type || !row_major(qkv)) {
    return 0;
  }
  CacheShape const c(k, heads_first);
  int const heads = heads_in(qkv, c.head_dim);
  if ((long long)heads <= 2LL * c.kv_heads || (long long)heads * c.head_dim > 1 << 30 || !angles_ok(positions, angles, qkv.dim[0], c.head_dim) || !has_dims(slots, {qkv.dim[0]}) ||
      slots.data_type != DT_INT32 || !row_major(slots) || qkv.data_ptr == k.data_ptr || qkv.data_ptr == v.data_ptr) {
    return 0;
  }
  return heads - 2 * c.kv_heads;
}

bool attention_ok(DTensor const &q, DTensor const &k, DTensor const &v, DTensor const &table, DTensor const &lengths, float scale,
                  int window, bool heads_first) {
  if (!caches_ok(k, v, heads_first) || q.data_type != k.data_type || !row_major(q) || window < 0 || !std::isfinite(scale)) {
    return false;
  }
  CacheShape const c(k, heads_first);
  int const heads = heads_in(q, c.head_dim);
  if (heads == 0 || heads % c.kv_heads != 0 || c.head_dim % 8 != 0 || c.head_dim > MI355_MAX_PAGED_HEAD_DIM) {
    return false;
  }
  // what mi355_paged_attention counts in 32 bits: places of a token, 16-byte steps into a cache, units of work of a sequence
  long long const new_tokens = table.num_dims == 2 && positive(table) ? q.dim[0] / table.dim[0] : 0;
  long long const keys = table.num_dims == 2 ? (long long)table.dim[1] * c.page_size : 0;
  if (new_tokens * heads > 1 << 29 || keys > 1 << 30 || (long long)heads * c.head_dim > INT_MAX || (unsigned long long)k.num_elements() / 8 >= UINT_MAX ||
      mi355::paged::too_many_units(c.kv_heads, new_tokens * (heads / c.kv_heads), keys)) {
    return false;
  }
  return positive(q) && table.num_dims == 2 && positive(table) && table.data_type == DT_INT32 && row_major(table) && has_dims(lengths, {table.dim[0]}) &&
         lengths.data_type == DT_INT32 && row_major(lengths) && q.dim[0] % table.dim[0] == 0 &&
         (long long)table.dim[1] * c.page_size <= 1 << 30 && (long long)(q.dim[0] / table.dim[0]) * heads <= 1 << 29;
}

// `t` as [rows, vocabulary] of `rows` rows: [sequences, per, vocabulary] or [sequences * per, vocabulary]
bool probabilities_ok(DTensor const &t, int sequences, int per) {
  bool const dims = t.num_dims == 3 ? t.dim[0] == sequences && t.dim[1] == per
                                    : t.num_dims == 2 && (long long)t.dim[0] == (long long)sequences * per;
  return dims && positive(t) && (half_type(t) || t.data_type == DT_FLOAT32) && row_major(t);
}

bool verify_ok(DTensor const &target, DTensor const *draft, DTensor const &tokens, DTensor const &uniforms) {
  if (tokens.num_dims != 2 || !positive(tokens) || tokens.dim[1] > INT_MAX / 2 || tokens.data_type != DT_INT32 || !row_major(tokens)) {
    return false;
  }
  int const sequences = tokens.dim[0], drafts = tokens.dim[1];
  return probabilities_ok(target, sequences, drafts + 1) &&
         (draft == nullptr || (probabilities_ok(*draft, sequences, drafts) && draft->data_type == target.data_type &&
                               draft->dim[draft->num_dims - 1] == target.dim[target.num_dims - 1])) &&
         has_dims(uniforms, {sequences, drafts + 1}) && uniforms.data_type == DT_FLOAT32 && row_major(uniforms);
}

std::vector<DTensor> verify_inputs(DTensor const &target, DTensor const *draft, DTensor const &tokens, DTensor const &uniforms) {
  std::vector<DTensor> in{target};
  if (draft != nullptr) {
    in.push_back(*draft);
  }
  in.push_back(tokens);
  in.push_back(uniforms);
  return in;
}

DTensor queries_of(DTensor const &qkv, int q_heads, int head_dim) {
  return qkv.num_dims == 3 ? tensor_of({qkv.dim[0], q_heads, head_dim}, qkv.data_type)
                           : tensor_of({qkv.dim[0], q_heads * head_dim}, qkv.data_type);
}

DTensor push(std::vector<KNOperator *> &ops, KNOperator *op, char const *what) {
  MIRAGE_CHECK(op != nullptr, what);
  ops.push_back(op);
  return op->output_tensors[0];
}

}  // namespace

bool is_decoding_op(KNOperatorType type) { return type >= KN_ROTARY_OP && type <= KN_VERIFY_DRAFTS_OP; }

bool Graph::keeps_inputs() const {
  for (KNOperator const *op : operators) {
    if (is_decoding_op(op->op_type)) {
      return true;
    }
  }
  return false;
}

KNDecodingOp::KNDecodingOp(KNOperatorType type, std::vector<DTensor> inputs) : KNOperator(type, std::move(inputs)) {}
KNDecodingOp::~KNDecodingOp() { release_outputs(); }

KNDecodingOp::operator json() const {
  json j;
  to_json(j, static_cast<KNOperator const &>(*this));
  return j;
}

bool KNDecodingOp::profile(ProfileResult &result) {
  if (without_kernel(*this) != nullptr) {
    result = ProfileResult::infinity();
    return false;
  }
  require_device("KNDecodingOp::profile");
  int const iters = 16;
  run();
  MI355_CALL(mi355_timer_start());
  for (int i = 0; i < iters; i++) {
    run();
  }
  float ms = 0.0f;
  MI355_CALL(mi355_timer_stop(&ms));
  result.run_time = ms / iters;
  return true;
}

// ---- rotary ------------------------------------------------------------------------------
KNOperator *Graph::create_rotary_op(DTensor const &x, DTensor const &positions, DTensor const &angles, bool interleaved) {
  return rotary_ok(x, positions, angles) && room_for(x) ? new KNRotaryOp(x, positions, angles, interleaved) : nullptr;
}

DTensor Graph::rotary(DTensor const &x, DTensor const &positions, DTensor const &angles, bool interleaved) {
  return push(operators, create_rotary_op(x, positions, angles, interleaved), "infeasible rotary");
}

KNRotaryOp::KNRotaryOp(DTensor const &x, DTensor const &positions, DTensor const &angles, bool _interleaved)
    : KNDecodingOp(KN_ROTARY_OP, {x, positions, angles}), interleaved(_interleaved) {
  MIRAGE_CHECK(rotary_ok(x, positions, angles), "rotary operands do not agree");
  adopt(this, tensor_of({x.dim[0], x.dim[1], x.dim[2]}, x.data_type));
}

void KNRotaryOp::run() const {
  DTensor const &x = input_tensors[0];
  long long const stride = (long long)x.dim[1] * x.dim[2];
  MI355_CALL(mi355_rotary(x.data_ptr, stride, output_tensors[0].data_ptr, stride, static_cast<int const *>(input_tensors[1].data_ptr),
                          static_cast<double const *>(input_tensors[2].data_ptr), x.dim[0], x.dim[1], x.dim[2],
                          input_tensors[2].dim[1], interleaved ? 1 : 0, x.data_type));
}

// ---- rotary_append -------------------------------------------------------------------------
KNOperator *Graph::create_rotary_append_op(DTensor const &qkv, DTensor const &positions, DTensor const &angles, DTensor const &slots,
                                           DTensor const &k_cache, DTensor const &v_cache, bool interleaved, bool heads_first) {
  int const q_heads = append_q_heads(qkv, positions, angles, slots, k_cache, v_cache, heads_first);
  return q_heads > 0 && room_for(queries_of(qkv, q_heads, k_cache.dim[3]))
             ? new KNRotaryAppendOp(qkv, positions, angles, slots, k_cache, v_cache, interleaved, heads_first)
             : nullptr;
}

DTensor Graph::rotary_append(DTensor const &qkv, DTensor const &positions, DTensor const &angles, DTensor const &slots,
                             DTensor const &k_cache, DTensor const &v_cache, bool interleaved, bool heads_first) {
  return push(operators, create_rotary_append_op(qkv, positions, angles, slots, k_cache, v_cache, interleaved, heads_first),
              "infeasible rotary_append");
}

KNRotaryAppendOp::KNRotaryAppendOp(DTensor const &qkv, DTensor const &positions, DTensor const &angles, DTensor const &slots,
                                   DTensor const &k_cache, DTensor const &v_cache, bool _interleaved, bool _heads_first)
    : KNDecodingOp(KN_ROTARY_APPEND_OP, {qkv, positions, angles, slots, k_cache, v_cache}), interleaved(_interleaved),
      heads_first(_heads_first) {
  int const q_heads = append_q_heads(qkv, positions, angles, slots, k_cache, v_cache, heads_first);
  MIRAGE_CHECK(q_heads > 0, "rotary_append operands do not agree");
  adopt(this, queries_of(qkv, q_heads, k_cache.dim[3]));
}

void KNRotaryAppendOp::run() const {
  DTensor const &qkv = input_tensors[0], &q = output_tensors[0];
  mi355_paged_cache const cache = cache_of(input_tensors[4], input_tensors[5], heads_first);
  int const heads = heads_in(qkv, cache.head_dim), q_heads = heads - 2 * cache.kv_heads;
  long long const stride = (long long)heads * cache.head_dim, q_stride = (long long)q_heads * cache.head_dim;
  auto const *base = static_cast<char const *>(qkv.data_ptr);
  size_t const size = get_datatype_size(qkv.data_type);
  MI355_CALL(mi355_rotary_append(base, stride, base + q_stride * size, stride,
                                 base + (q_stride + (long long)cache.kv_heads * cache.head_dim) * size, stride, q.data_ptr, q_stride,
                                 static_cast<int const *>(input_tensors[1].data_ptr),
                                 static_cast<double const *>(input_tensors[2].data_ptr),
                                 static_cast<int const *>(input_tensors[3].data_ptr), &cache, qkv.dim[0], q_heads,
                                 input_tensors[2].dim[1], interleaved ? 1 : 0));
}

// ---- paged_attention -------------------------------------------------------------------------
KNOperator *Graph::create_paged_attention_op(DTensor const &q, DTensor const &k_cache, DTensor const &v_cache, DTensor const &table,
                                             DTensor const &lengths, float scale, int window, bool heads_first) {
  return attention_ok(q, k_cache, v_cache, table, lengths, scale, window, heads_first) && room_for(q)
             ? new KNPagedAttentionOp(q, k_cache, v_cache, table, lengths, scale, window, heads_first)
             : nullptr;
}

DTensor Graph::paged_attention(DTensor const &q, DTensor const &k_cache, DTensor const &v_cache, DTensor const &table,
                               DTensor const &lengths, float scale, int window, bool heads_first) {
  return push(operators, create_paged_attention_op(q, k_cache, v_cache, table, lengths, scale, window, heads_first),
              "infeasible paged_attention");
}

KNPagedAttentionOp::KNPagedAttentionOp(DTensor const &q, DTensor const &k_cache, DTensor const &v_cache, DTensor const &table,
                                       DTensor const &lengths, float _scale, int _window, bool _heads_first)
    : KNDecodingOp(KN_PAGED_ATTENTION_OP, {q, k_cache, v_cache, table, lengths}), scale(_scale), window(_window),
      heads_first(_heads_first) {
  MIRAGE_CHECK(attention_ok(q, k_cache, v_cache, table, lengths, scale, window, heads_first), "paged_attention operands do not agree");
  adopt(this, queries_of(q, heads_in(q, k_cache.dim[3]), k_cache.dim[3]));
}

void KNPagedAttentionOp::run() const {
  DTensor const &q = input_tensors[0], &table = input_tensors[3];
  mi355_paged_cache const cache = cache_of(input_tensors[1], input_tensors[2], heads_first);
  int const q_heads = heads_in(q, cache.head_dim);
  long long const stride = (long long)q_heads * cache.head_dim;
  MI355_CALL(mi355_paged_attention(q.data_ptr, stride, output_tensors[0].data_ptr, stride, &cache,
                                   static_cast<int const *>(table.data_ptr), table.dim[1],
                                   static_cast<int const *>(input_tensors[4].data_ptr), table.dim[0], q.dim[0] / table.dim[0], q_heads,
                                   scale, window));
}

// ---- verify_drafts -----------------------------------------------------------------------------
KNOperator *Graph::create_verify_drafts_op(DTensor const &target, DTensor const *draft, DTensor const &tokens,
                                           DTensor const &uniforms) {
  if (!verify_ok(target, draft, tokens, uniforms)) {
    return nullptr;
  }
  size_t const b = (size_t)tokens.dim[0], all = b * (tokens.dim[1] + 1);
  return room_for({4 * b, 4 * all}, {2 * b, 2 * all}) ? new KNVerifyDraftsOp(target, draft, tokens, uniforms) : nullptr;
}

std::vector<DTensor> Graph::verify_drafts(DTensor const &target, DTensor const *draft, DTensor const &tokens,
                                          DTensor const &uniforms) {
  push(operators, create_verify_drafts_op(target, draft, tokens, uniforms), "infeasible verify_drafts");
  return operators.back()->output_tensors;
}

KNVerifyDraftsOp::KNVerifyDraftsOp(DTensor const &target, DTensor const *draft, DTensor const &tokens, DTensor const &uniforms)
    : KNDecodingOp(KN_VERIFY_DRAFTS_OP, verify_inputs(target, draft, tokens, uniforms)) {
  MIRAGE_CHECK(verify_ok(target, draft, tokens, uniforms), "verify_drafts operands do not agree");
  adopt(this, tensor_of({tokens.dim[0]}, DT_INT32));
  adopt(this, tensor_of({tokens.dim[0], tokens.dim[1] + 1}, DT_INT32));
}

void KNVerifyDraftsOp::run() const {
  bool const certain = input_tensors.size() == 3;
  DTensor const &target = input_tensors[0], &tokens = input_tensors[certain ? 1 : 2], &uniforms = input_tensors[certain ? 2 : 3];
  MI355_CALL(mi355_verify_drafts(target.data_ptr, certain ? nullptr : input_tensors[1].data_ptr,
                                 static_cast<int const *>(tokens.data_ptr), static_cast<float const *>(uniforms.data_ptr),
                                 static_cast<int *>(output_tensors[0].data_ptr), static_cast<int *>(output_tensors[1].data_ptr),
                                 tokens.dim[0], tokens.dim[1], target.dim[target.num_dims - 1], target.data_type));
}

}  // namespace kernel
}  // namespace mirage

// ---- C facade (tensor handles as in c_api.cc; null / -1: infeasible) ---------------------------------
extern "C" {

using mirage::kernel::DTensor;
using mirage::kernel::Graph;
using mirage::kernel::KNOperator;

static void *keep(Graph *g, KNOperator *op) {
  if (op == nullptr) {
    return nullptr;
  }
  g->operators.push_back(op);
  return &op->output_tensors[0];
}
static DTensor const &at(void *t) { return *static_cast<DTensor const *>(t); }

void *mirage_graph_rotary(void *g, void *x, void *positions, void *angles, int interleaved) {
  auto *G = static_cast<Graph *>(g);
  return keep(G, G->create_rotary_op(at(x), at(positions), at(angles), interleaved != 0));
}

void *mirage_graph_rotary_append(void *g, void *qkv, void *positions, void *angles, void *slots, void *k_cache, void *v_cache,
                                 int interleaved, int heads_first) {
  auto *G = static_cast<Graph *>(g);
  return keep(G, G->create_rotary_append_op(at(qkv), at(positions), at(angles), at(slots), at(k_cache), at(v_cache),
                                            interleaved != 0, heads_first != 0));
}

void *mirage_graph_paged_attention(void *g, void *q, void *k_cache, void *v_cache, void *table, void *lengths, float scale,
                                   int window, int heads_first) {
  auto *G = static_cast<Graph *>(g);
  return keep(G, G->create_paged_attention_op(at(q), at(k_cache), at(v_cache), at(table), at(lengths), scale, window,
                                              heads_first != 0));
}

// outputs[0] = accepted, outputs[1] = tokens; draft may be null
int mirage_graph_verify_drafts(void *g, void *target, void *draft, void *tokens, void *uniforms, void **outputs) {
  auto *G = static_cast<Graph *>(g);
  if (keep(G, G->create_verify_drafts_op(at(target), static_cast<DTensor const *>(draft), at(tokens), at(uniforms))) == nullptr) {
    return -1;
  }
  outputs[0] = &G->operators.back()->output_tensors[0];
  outputs[1] = &G->operators.back()->output_tensors[1];
  return 0;
}

}  // extern "C"
