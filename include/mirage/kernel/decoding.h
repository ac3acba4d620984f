// Kernel-level operators of a decoding step that keeps its keys and values in a paged cache (extensions of this
// backend, not in the reference).  Two tensors [pages, page_size, kv_heads, head_dim], or [pages, kv_heads, page_size,
// head_dim] with heads_first, hold the keys and the values; a sequence's page table names its pages in order, and a
// slot is page * page_size + place in the page.  Values are fp16 or bf16, indices DT_INT32, every tensor is row-major.
//
// They have no image in the fingerprint ring (angles, the largest of a row, comparisons with random numbers):
// fingerprint() returns false, and a graph that holds one is refused by the fingerprinting of whole graphs.
#pragma once

#include "mirage/kernel/operator.h"

namespace mirage {
namespace kernel {

// Whether `type` is one of the operators below.
bool is_decoding_op(mirage::type::KNOperatorType type);

class KNDecodingOp : public KNOperator {
public:
  KNDecodingOp(mirage::type::KNOperatorType type, std::vector<DTensor> inputs);
  ~KNDecodingOp();
  // false, and nothing run, where a caller has declared one of the tensors column-major (a layout search does not)
  bool profile(ProfileResult &result) override;
  bool fingerprint(void) override { return false; }
  operator json() const override;
  virtual void run(void) const = 0;  // one execution on the backend stream, no synchronisation
};

// Rotary positions of x [tokens, heads, head_dim]: the pair i of a head, (x[i], x[i + R/2]) or, interleaved,
// (x[2i], x[2i + 1]), is turned by the angle positions[token] * angles[0][i] and scaled by angles[1][i]; elements from
// R on stay.  positions [tokens]; angles [2, R/2], DT_DOUBLE.  Any scaling for long contexts is in the angles.
class KNRotaryOp : public KNDecodingOp {
public:
  KNRotaryOp(DTensor const &x, DTensor const &positions, DTensor const &angles, bool interleaved);
  void run(void) const override;
  bool interleaved;
};

// The same for the queries and keys of one projection qkv, [tokens, q_heads + 2 kv_heads, head_dim] or
// [tokens, (q_heads + 2 kv_heads) head_dim]: the queries are the result, the keys and the values are written into the
// caches, IN PLACE, at slots[token].  A negative slot, or one past the cache, stores nothing.  The slots of one call
// differ: of one that is named twice, any element may come from either token.
class KNRotaryAppendOp : public KNDecodingOp {
public:
  KNRotaryAppendOp(DTensor const &qkv, DTensor const &positions, DTensor const &angles, DTensor const &slots,
                   DTensor const &k_cache, DTensor const &v_cache, bool interleaved, bool heads_first);
  void run(void) const override;
  bool interleaved, heads_first;
};

// softmax(scale q K^T) V of the new tokens of every sequence.  q [sequences * new, q_heads, head_dim] or
// [sequences * new, q_heads * head_dim], a sequence's tokens in a row; table [sequences, most pages of one]; lengths
// [sequences], the new tokens (whose keys are in the cache already) among them: new token t sees the keys before
// L = length - (new - 1 - t), of these the last `window` where that is not 0.  Query head h reads key-value head
// h / (q_heads / kv_heads).  A row that sees no key, or only scores of minus infinity, is zeros; a page number outside the cache holds no keys; a length
// past the table counts as the table's.  What lies in places that a row does not see never reaches it; a seen value that is
// infinite makes its column infinite, NaN beside one of the other sign (either, where its weight is below 2^-30 of the row's
// greatest); a NaN makes it NaN.
class KNPagedAttentionOp : public KNDecodingOp {
public:
  KNPagedAttentionOp(DTensor const &q, DTensor const &k_cache, DTensor const &v_cache, DTensor const &table,
                     DTensor const &lengths, float scale, int window, bool heads_first);
  void run(void) const override;
  float scale;
  int window;
  bool heads_first;
};

// Speculative sampling's decision.  target [sequences, drafts + 1, vocabulary] (or its first two dimensions as one):
// probabilities, fp16, bf16 or DT_FLOAT32, after each draft taken so far; draft likewise [sequences, drafts,
// vocabulary], those the drafts were drawn from, or none: they were certain; tokens [sequences, drafts], a negative one
// (or one past the vocabulary) ends a sequence's drafts; uniforms [sequences, drafts + 1], DT_FLOAT32, in [0, 1).
// Draft i is taken while uniforms[i] * draft[i][token] < target[i][token].  The token after them is drawn by the last
// uniform from max(target - draft, 0) (certain: from target without the token) if one was refused, from target if none
// was left, the lowest index whose sum of weights passes its share; from target too where the differences are all zero.
// Results: accepted [sequences], and tokens [sequences, drafts + 1]: those taken, the drawn one (-1: target has no
// weight), then -1.
class KNVerifyDraftsOp : public KNDecodingOp {
public:
  KNVerifyDraftsOp(DTensor const &target, DTensor const *draft, DTensor const &tokens, DTensor const &uniforms);
  void run(void) const override;
};

}  // namespace kernel
}  // namespace mirage
