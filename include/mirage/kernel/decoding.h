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

// Attention of a tree of drafted tokens of every sequence: as paged attention, but of the new tokens a row sees its own node
// of the tree and that one's ancestors.  parents [sequences, nodes], nodes = new tokens of a sequence, up to 1024: the node
// that node i follows, one before it; -1: it follows the sequence itself.  The keys of node i are at place
// length - nodes + i.  A node with any other parent, or a place below zero, is not there, nor is what follows it: its row is
// zeros and no row sees its key (so fewer drafts are padded).  Values, scores and page numbers that are out of order: as in
// paged attention.  Where nodes times the query heads of a key-value head are more than 16, weights are rounded once to the values' type
// (in paged attention to 2^-16), and the sum of weights is that of the rounded ones: as much error again as the result's own rounding.
class KNTreeAttentionOp : public KNDecodingOp {
public:
  KNTreeAttentionOp(DTensor const &q, DTensor const &k_cache, DTensor const &v_cache, DTensor const &table, DTensor const &lengths,
                    DTensor const &parents, float scale, bool heads_first);
  void run(void) const override;
  float scale;
  bool heads_first;
};

// Attention within a window, and to the first tokens of the sequence: as paged attention, but new token t sees the keys j <
// L = length - (new - 1 - t) with j >= L - window (all, where window is 0) or j < sinks.  One new token of every sequence, whole
// prompts, or anything between; with starts [sequences + 1], ascending from 0, sequence b's new tokens are the rows starts[b] to
// starts[b + 1] - 1 of q, and rows from the last of them on are left as they were; without, every sequence has as many.  Weights are
// rounded as in attention of trees, with starts whatever the rows.
class KNWindowAttentionOp : public KNDecodingOp {
public:
  KNWindowAttentionOp(DTensor const &q, DTensor const &k_cache, DTensor const &v_cache, DTensor const &table, DTensor const &lengths,
                      DTensor const *starts, float scale, int window, int sinks, bool heads_first);
  void run(void) const override;
  float scale;
  int window, sinks;
  bool heads_first;
};

// Of logits [rows, vocabulary] (or their first two dimensions as one; fp16, bf16 or DT_FLOAT32), times a scale above zero, as
// a distribution: the log probabilities of tokens [rows] or [rows, asked] (minus infinity for one outside the vocabulary), of
// the same shape; its entropy [rows]; and for top > 0 the `top` most probable tokens of every row, of equal logits the lower
// index first, [rows, top], behind their log probabilities.  Up to 64; a token without probability is none of them: -1, minus
// infinity.  Everything in natural units, DT_FLOAT32.  A row of minus infinities has log probabilities of minus infinity,
// entropy zero and no top tokens; one with a NaN or plus infinity NaN for all numbers, and -1.
class KNLogProbabilitiesOp : public KNDecodingOp {
public:
  KNLogProbabilitiesOp(DTensor const &logits, DTensor const &tokens, int top, float scale);
  void run(void) const override;
  int top;
  float scale;
};

}  // namespace kernel
}  // namespace mirage
