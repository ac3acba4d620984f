// Attention of blocks of rows over a paged key-value cache: whole prompts and chunks of them within a window, and trees of
// drafted tokens.
//
// o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q . k_j, over the keys a row sees, in one pass with a running
// maximum.  A row is a new token and one of the query heads that share a key-value head, so that these heads share its keys too.
// * A workgroup has 128 rows, a wavefront 32 of them; tiles of keys and values come from the pages straight into LDS, the next
//   while one is worked on: one barrier a tile.
// * Scores are made transposed, S^T = K Q^T, by products of 32 x 32 x 16: a lane then has half the weights of one row, of the
//   keys that it has as the operand of O^T = V^T P^T if values are read in that order.  No weight changes lanes.
// * Keys are counted as the block sees them: the first `kept` of the sequence, then those from `first` on, in one run without a gap;
//   where up to 2048 of the run lie is looked up at once and kept in LDS.
// * Weights are rounded to the values' type once, and added up as rounded: an error of as much again as rounding the result makes, at
//   two thirds of the matrix products that weights in two words would take.  (The ABI says so.)
// * Blocks that leave compute units without work are cut along their keys (of trees so that all parts are alike), and joined by a second
//   kernel in the order of the keys, so that results do not depend on who comes first.
//
// Measured (8 key-value heads of 4 query heads of 128, bf16): 555 to 597 us of one prompt of 8192 tokens (550 GFLOP, 920 to 990 TFLOP/s), 164 to 177 within a
// window of 1024 (129 GFLOP, 730 to 790 TFLOP/s); a large matrix product reaches 1270.  What bounds it are the two wavefronts of a SIMD taking
// turns: matrix instructions fill 37 % of its cycles and vector instructions, exponentials nearly half of them, 48 %.
#pragma once

#include "mi355_kernels/attention_blocks_units.h"
#include "paged_attention.h"

namespace mi355 {
namespace blocks {

using paged::exp2_fast;
using paged::quotient;
using paged::uintx4;
using paged::Vec;

struct BlockParams {
  void const *q, *k, *v;
  void *out;
  long long q_stride, out_stride;
  uint32_t page_step, token_step, head_step;  // in 16 bytes
  int const *table, *lengths;
  int const *starts;   // of ragged batches, or null
  int const *parents;  // of trees
  int pages, page_size, head_dim, table_width, sequences, tokens, new_tokens, group, kv_heads, window, sinks;
  int row_blocks;  // of a sequence, where all have new_tokens
  int blocks;      // of all sequences, at most
  int slots;       // workgroups that the chip holds together
  int splits;      // parts that the keys of a block are cut into, at most
  int least;       // keys of a part, at least: whole tiles
  float *parts;    // of every block and part: sums as the lanes hold them, then reference and sum of weights of its rows
  unsigned page_magic, group_magic;
  uint32_t q_keep, q_flip;
  float scale;
};

int launch_f16(BlockParams const &P, bool tree);
int launch_bf16(BlockParams const &P, bool tree);

typedef float floatx16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ floatx16 mfma(Vec<_Float16>::x8 a, Vec<_Float16>::x8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma(Vec<__bf16>::x8 a, Vec<__bf16>::x8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Where 16-byte chunk `chunk` of row `row` lies in a tile of C chunks a row.  There are 64 banks of 4 bytes, sixteen chunks: sixteen rows in
// a row that read the same chunk (keys) meet them all, and so do four rows that read four chunks in a row (values).
template <int C>
__device__ __forceinline__ int turn_of(int row) {
  return C == 8 || C == 24 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : C == 12 ? row >> 2 & 3 : (row & 3) << 2 | (row >> 2 & 3);
}
template <int C>
__device__ __forceinline__ int place_of(int row, int chunk) {
  int const turn = turn_of<C>(row);
  if constexpr ((C & (C - 1)) == 0) {
    return chunk ^ turn;
  }
  int const at = chunk + turn;
  return at >= C ? at - C : at;
}
template <int C>
__device__ __forceinline__ int chunk_at(int row, int place) {
  int const turn = turn_of<C>(row);
  if constexpr ((C & (C - 1)) == 0) {
    return place ^ turn;
  }
  int const chunk = place - turn;
  return chunk < 0 ? chunk + C : chunk;
}

// x[l] op x[l ^ 32] in every lane
template <class Op>
__device__ __forceinline__ float over_halves(float x, Op op) {
  float a = x, b = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return op(a, b);
}

// sum + the eight elements: two to an instruction
__device__ __forceinline__ float sum_of(Vec<_Float16>::x8 p, float sum) {
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    sum = __builtin_amdgcn_fdot2(pair{p[i], p[i + 1]}, pair{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
  }
  return sum;
}
__device__ __forceinline__ float sum_of(Vec<__bf16>::x8 p, float sum) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    sum = __builtin_amdgcn_fdot2_f32_bf16(pair{p[i], p[i + 1]}, pair{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
  }
  return sum;
}

__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1); }

constexpr int kThreads = 256, kWaves = 4;
template <int DP>
constexpr int kKeys = DP == 192 ? 32 : 64;  // of a tile
template <int DP, bool TREE>
constexpr int kStepsOf = DP != 96 ? 2048 : (TREE ? 512 : 1024);  // keys of a run whose places a workgroup holds in LDS (96: three workgroups fit)
template <int DP>
constexpr int tile_bytes() { return kKeys<DP> * DP * 2; }
template <int DP, bool TREE>
constexpr int lds_bytes() { return 4 * tile_bytes<DP>() + 4 * kStepsOf<DP, TREE> + kStepsOf<DP, TREE> / 8 + 32 + (TREE ? 2 * MI355_MAX_TREE_NODES : 0); }
// Workgroups that a compute unit holds, its registers and LDS (of trees with heads up to 64: three, 45 us, where two are asked for, 50; 4 x 4 heads x up to
// 16384 keys, 512 rows).  Heads of 256: one, of tiles of 64 keys (one prompt of 8192 tokens, 32 heads, a window
// of 1024: 440 us; two of tiles of 32, with registers spilled, 459).
template <int DP>
constexpr int kPerUnit = DP <= 96 ? 3 : DP <= 192 ? 2 : 1;

// The rows of a block and the keys that any of them sees.
struct Block {
  int sequence, row_of_q, new_tokens, row0, rows, length;
  int kept, shift, end;  // key j of the run is key j of the sequence below `kept`, j + shift from there on
  bool is;
};
template <bool TREE>
__device__ __forceinline__ Block block_of(BlockParams const &P, int block) {
  int const lane = threadIdx.x % 64;
  Block b{};
  if (P.starts == nullptr) {
    b.sequence = block / P.row_blocks;
    block -= b.sequence * P.row_blocks;
    b.row_of_q = b.sequence * P.new_tokens;
    b.new_tokens = P.new_tokens;
  } else {
    // A sequence's blocks are numbered from before(its first token) + its own number on, which leaves room for all of them: the last sequence
    // that begins no later than the block is found among 64 at a time.
    auto before = [&](int token) { return token * P.group / kRows; };
    int first = 0;
    for (int n = P.sequences, step = 0; step != 1;) {
      step = (n + 63) / 64;
      int const at = lane * step < n ? first + lane * step : first;
      auto start = [&](int i) {
        int const s = P.starts[i];
        return s < 0 ? 0 : (s < P.tokens ? s : P.tokens);
      };
      int const from = start(at), to = start(at + 1);
      uint64_t const begun = __ballot(lane * step < n && before(from) + at <= block);
      if (begun == 0) {
        return b;
      }
      int const which = 63 - __builtin_clzll(begun);
      first += which * step;
      n = n - which * step < step ? n - which * step : step;
      b.row_of_q = __builtin_amdgcn_readlane(from, which);
      b.new_tokens = __builtin_amdgcn_readlane(to, which) - b.row_of_q;
    }
    b.sequence = first;
    int const its = b.new_tokens > 0 ? (b.new_tokens * P.group + kRows - 1) / kRows : 0;
    block -= before(b.row_of_q) + first;
    if (block >= its) {
      return b;
    }
    // (as in_order, sequence by sequence: 199 -> 178 us of four chunks of up to 3000 behind up to 7001 keys, 5 x 3 heads of 80)
    block = P.window == 0 ? its - 1 - block : block;
  }
  b.is = true;
  int const R = b.new_tokens * P.group, most = P.table_width * P.page_size, told = P.lengths[b.sequence];
  b.row0 = block * kRows;
  b.rows = R - b.row0 < kRows ? R - b.row0 : kRows;
  b.length = told < 0 ? 0 : (told < most ? told : most);
  int const before = b.length - b.new_tokens + 1;  // what the first new token sees, without a window
  int to = TREE ? b.length : before + quotient(b.row0 + b.rows - 1, P.group, P.group_magic);
  to = to < 0 ? 0 : to;
  int first = !TREE && P.window != 0 ? before + quotient(b.row0, P.group, P.group_magic) - P.window : 0;
  first = first < 0 ? 0 : first;
  b.kept = P.sinks < first ? P.sinks : first;
  b.shift = first - b.kept;
  b.end = to - b.shift;
  return b;
}

// the parents of its nodes, -2 in the place of any that is none
__device__ __forceinline__ void fetch_tree(BlockParams const &P, Block const &b, short *tree) {
  for (int i = threadIdx.x; i < b.new_tokens; i += kThreads) {
    int const p = P.parents[(long long)b.sequence * b.new_tokens + i];
    tree[i] = (short)(p >= -1 && p < i ? p : -2);
  }
}

// Without a window the last blocks of sequences have the most keys: these come first, and the short ones where workgroups are left without work.
// (614 -> 555 us of one prompt of 8192 tokens, 8 x 4 heads of 128, 179 -> 161 of 4096, where the end waited for long ones.)
template <bool TREE>
__device__ __forceinline__ int in_order(BlockParams const &P, int item) {
  if (TREE || P.window != 0 || P.starts != nullptr) {
    return item;
  }
  int const rank = item / P.sequences;
  return (item - rank * P.sequences + 1) * P.row_blocks - 1 - rank;
}

// A row of it: the keys of the run below `always`, and those from `least` up to `limit`; of a tree, those below `limit` (below zero:
// none) and the token's and its ancestors'.
struct Row {
  int row, token, limit, least, always;
};
template <bool TREE>
__device__ __forceinline__ Row row_of(BlockParams const &P, Block const &b, int in_block, short const *tree) {
  Row r{b.row0 + in_block, 0, 0, 0, 0};
  r.token = quotient(in_block < b.rows ? r.row : b.row0 + b.rows - 1, P.group, P.group_magic);
  int const context = b.length - b.new_tokens;
  if (in_block < b.rows) {
    r.limit = TREE ? context : context + 1 + r.token - b.shift;
    r.least = !TREE && P.window != 0 ? r.limit - P.window : 0;
    r.always = P.sinks < r.limit ? P.sinks : r.limit;
  }
  if constexpr (TREE) {  // whether every ancestor is there
    int at = in_block < b.rows && context + r.token >= 0 ? r.token : -2;
    while (__any(at >= 0)) {
      if (at >= 0) {
        int const p = tree[at];
        at = p < 0 || context + p >= 0 ? p : -2;
      }
    }
    r.limit = at == -1 ? (r.limit < 0 ? 0 : r.limit) : -1;
  }
  if (in_block >= b.rows) {  // no tile is masked for rows that are not there (131 -> 127 us of ragged chunks)
    r.limit = INT_MAX;
    r.least = 0;
  }
  return r;
}
// weights are at most 2^(bias + kSlack)
constexpr float kSlack = 6.0f;
// Weights are 2^(scale s + (bias - scale ref)) with one rounding of what is in brackets, which all weights have alike; from a reference of 2^25 on it would take them
// past the types' ends.  Above this the difference of scores comes first.
constexpr float kLarge = 0x1p20f;
template <class T>
__device__ __forceinline__ float bias_of(int keys) {
  return std::is_same<T, _Float16>::value ? 9.0f : (float)(__builtin_clz((unsigned)keys | 1u) - 33) - kSlack;
}

// How the blocks of a batch of trees are cut along their keys: a tree's all into as many parts as leave each at most `run` tiles, with the
// least run for which the parts of all are no more than the workgroups that the chip holds together (P.slots, and the launch's).
struct Cut {
  int sequence, parts, before;  // a sequence, the parts of each of its blocks, the workgroups of the sequences before it
};
template <int DP>
__device__ __forceinline__ Cut cut_of(BlockParams const &P, int work, int sequence) {  // of the sequence with that workgroup, or of that one (work -1)
  int const lane = threadIdx.x % 64, each = P.row_blocks * P.kv_heads, most = P.table_width * P.page_size;
  auto tiles_of = [&](int i) {
    int const told = i < P.sequences ? P.lengths[i] : 0, length = told < 0 ? 0 : (told < most ? told : most);
    int const tiles = (length + kKeys<DP> - 1) / kKeys<DP>;
    return tiles < 1 ? 1 : (tiles < 1 << 20 ? tiles : 1 << 20);  // (their sum over fewer blocks than slots fits 32 bits)
  };
  int const own = tiles_of(lane);
  auto total = [&](auto value) {
    int x = lane < P.sequences ? value(own) : 0;
    for (int i = lane + 64; i < P.sequences; i += 64) {
      x += value(tiles_of(i));
    }
    return __builtin_amdgcn_readlane(paged::wave_upto(x), 63) * each;
  };
  int run = (total([](int tiles) { return tiles; }) + P.slots - 1) / P.slots;
  run = run < P.least / kKeys<DP> ? P.least / kKeys<DP> : run;
  auto parts_of = [&](int tiles) { return (int)(((unsigned)tiles + run - 1) / (unsigned)run); };
  while (total(parts_of) > P.slots) {
    run += 1 + run / 16;
  }
  Cut cut{-1, 0, 0};
  for (int base = 0; base < P.sequences; base += 64) {
    int const i = base + lane, parts = i < P.sequences ? parts_of(base == 0 ? own : tiles_of(i)) : 0, upto = paged::wave_upto(parts) * each;
    uint64_t const past = work >= 0 ? __ballot(cut.before + upto > work) : (sequence < base + 64 ? 1ull << (sequence - base) : 0);
    if (past != 0) {
      int const at = __builtin_ctzll(past);
      cut.sequence = base + at;
      cut.parts = __builtin_amdgcn_readlane(parts, at);
      cut.before += __builtin_amdgcn_readlane(upto - parts * each, at);
      return cut;
    }
    cut.before += __builtin_amdgcn_readlane(upto, 63);
  }
  return cut;
}
// Any other block is cut into as many parts as all may have, of P.least keys or more.
__device__ __forceinline__ int parts_of(BlockParams const &P, Block const &b) {
  int const most = b.end / P.least;
  return most < 1 ? 1 : (most < P.splits ? most : P.splits);
}
// of a block's part
template <int DP>
constexpr int part_floats() { return kRows * (DP + 2); }

// What sums are scaled by at least where there may be infinities among them: as good as zero, but zero times an infinity is NaN.
constexpr float kNone = 0x1p-126f;
// Adds the values of a tile that are infinite or NaN to the rows that see their keys (of both halves' lanes, a bit each), whatever the weights, and leaves
// zeros in their places.  All wavefronts do; `keys` are two words of LDS.
template <class T, int DP>
__device__ __forceinline__ void add_wild(unsigned char *v_tile, uint32_t *keys, uint64_t seen, floatx16 (&acc)[DP / 32]) {
  constexpr int C = DP / 8, LOADS = kKeys<DP> * C / kThreads;
  constexpr uint32_t top = Vec<T>::exponent;
  typedef typename Vec<T>::x4 x4;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // (what is made of it here is not to be kept through the loop over tiles)
  int const h = tid % 64 / 32;
  auto is_wild = [](uint32_t x) { return (x & top) == top || (x & top << 16) == top << 16; };
  if (tid < 2) {
    keys[tid] = 0;
  }
  __syncthreads();
  for (int i = 0; i < LOADS; i++) {
    int const n = kThreads * i + tid, its = n / C;
    uintx4 const x = *reinterpret_cast<uintx4 const *>(v_tile + 16 * n);
    if (is_wild(x[0]) || is_wild(x[1]) || is_wild(x[2]) || is_wild(x[3])) {
      __hip_atomic_fetch_or(keys + its / 32, 1u << its % 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
  __syncthreads();
  uint64_t const all = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)keys[1]) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)keys[0]);
  if (all == 0) {
    return;
  }
  for (uint64_t left = all; left != 0; left &= left - 1) {
    int const j = __builtin_ctzll(left);
    bool const sees = (seen >> j & 1) != 0;
#pragma unroll
    for (int d = 0; d < DP / 32; d++) {
#pragma unroll
      for (int four = 0; four < 4; four++) {
        x4 const x = *reinterpret_cast<x4 const *>(v_tile + j * (2 * DP) + 16 * place_of<C>(j, 4 * d + four) + 8 * h);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float const value = static_cast<float>(x[e]);
          acc[d][4 * four + e] += sees && !(__builtin_fabsf(value) < INFINITY) ? value : 0.0f;
        }
      }
    }
  }
  __syncthreads();
  for (int i = 0; i < LOADS; i++) {
    uintx4 *const place = reinterpret_cast<uintx4 *>(v_tile + 16 * (kThreads * i + tid));
    uintx4 x = *place;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      x[w] &= ((x[w] & top) == top ? 0u : 0xffffu) | ((x[w] & top << 16) == top << 16 ? 0u : 0xffff0000u);
    }
    *place = x;
  }
  __syncthreads();
}

template <class T, int DP, bool TREE>
__global__ __launch_bounds__(kThreads, kPerUnit<DP>) void attention_blocks_kernel(BlockParams const P) {
  fetch_kernel_arguments<sizeof(BlockParams), 0>();  // (gridDim is not read: no word behind them is the launch's)
  constexpr int KT = kKeys<DP>, G = KT / 32, C = DP / 8, LOADS = KT * C / kThreads, KK = DP / 16, DB = DP / 32, kSteps = kStepsOf<DP, TREE>;
  typedef typename Vec<T>::x8 x8;
  typedef typename Vec<T>::x4 x4;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  uint64_t *const exist = reinterpret_cast<uint64_t *>(lds + 4 * tile_bytes<DP>());
  uint32_t *const steps = reinterpret_cast<uint32_t *>(exist + kSteps / 64);
  uint32_t *const wild = steps + kSteps;  // for each wavefront whether its rows have sums that are not finite; keys of a tile with such values, a bit each
  short *const tree = reinterpret_cast<short *>(wild + 8);
  int const tid = threadIdx.x, lane = tid % 64, wave = tid / 64, h = lane / 32, c = lane % 32;
  uint32_t const lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void const *)lds;

  // the block and its part: key-value heads side by side (eight of them lie on an XCD each, with the keys that its blocks share)
  int const kv = (int)blockIdx.x % P.kv_heads;
  int item = (int)blockIdx.x / P.kv_heads, split = 0, parts = 1;
  bool const dealt = TREE && P.sequences > 1;  // parts are, to blocks of different lengths
  if (P.splits > 1) {
    if (dealt) {
      Cut const cut = cut_of<DP>(P, blockIdx.x, 0);
      if (cut.sequence < 0) {
        return;
      }
      int const rest = ((int)blockIdx.x - cut.before) / P.kv_heads;
      parts = cut.parts;
      split = rest / P.row_blocks;
      item = cut.sequence * P.row_blocks + rest % P.row_blocks;
    } else {
      split = item / P.blocks;
      item -= split * P.blocks;
    }
  }
  Block const b = block_of<TREE>(P, in_order<TREE>(P, item));
  if (P.splits > 1 && !dealt) {
    parts = parts_of(P, b);
  }
  if (!b.is || split >= parts) {
    return;
  }
  if constexpr (TREE) {
    fetch_tree(P, b, tree);
    __syncthreads();
  }
  int const context = b.length - b.new_tokens, kept = b.kept, shift = b.shift;
  int begin = 0, end = b.end;
  if (parts > 1) {
    int const tiles = (b.end + KT - 1) / KT;
    begin = (int)((long long)tiles * split / parts) * KT;
    end = (int)((long long)tiles * (split + 1) / parts) * KT;
    end = end < b.end ? end : b.end;
  }

  Row const r = row_of<TREE>(P, b, 32 * wave + c, tree);
  bool const is_row = 32 * wave + c < b.rows;
  x8 q[KK];
  {
    T const *const from = static_cast<T const *>(P.q) + (long long)(b.row_of_q + r.token) * P.q_stride +
                          (long long)(kv * P.group + (is_row ? r.row - r.token * P.group : 0)) * P.head_dim;
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
      int const d = 16 * kk + 8 * h;
      uintx4 x = {0, 0, 0, 0};
      if (is_row && d < P.head_dim) {
        x = *reinterpret_cast<uintx4 const *>(from + d);
      }
#pragma unroll
      for (int w = 0; w < 4; w++) {
        x[w] = (x[w] & P.q_keep) ^ P.q_flip;
      }
      q[kk] = __builtin_bit_cast(x8, x);
    }
  }

  floatx16 acc[DB];
  float ref, base, sum;
  // The reference follows the maximum only where weights would pass 2^(bias + kSlack), so that sums are seldom scaled.  fp16: small ones stay
  // above the type's end.  bf16: as values reach the end of 32 bits themselves, n weights add up to less than 1/2.
  float const bias = bias_of<T>(b.end);
  uint64_t const k_base = reinterpret_cast<uint64_t>(P.k) + 16ull * kv * P.head_step, v_base = reinterpret_cast<uint64_t>(P.v) + 16ull * kv * P.head_step;
  int const *const table = P.table + (long long)b.sequence * P.table_width;

  // The chunk of its key or value that this thread loads to each of its places.  Past the head's end values have their last one again, of which no result
  // is taken, keys zeros: queries are zero there, but zero times an infinity is not.  (Leaving such places zero and not loading them took longer: 90.5 us of
  // 64 single tokens, ragged, 5 x 3 heads of 80 x up to 7001 keys, so 88.1.)
  uint32_t chunk_of[LOADS];
  bool real[LOADS];
  bool const padded = P.head_dim < DP;
#pragma unroll
  for (int i = 0; i < LOADS; i++) {
    int const n = kThreads * i + tid, chunk = chunk_at<C>(n / C, n % C), last = P.head_dim / 8 - 1;
    chunk_of[i] = chunk < last ? chunk : last;
    real[i] = chunk <= last;
  }

  // A weight of zero does not keep an infinity or NaN among the values out of a sum, and looking for them in every tile that not all rows see would take too long:
  // where a sum comes out as none of the finite numbers the workgroup starts again with care, and each tile's are added to the rows that see them by
  // themselves, and zero from then on.  (One infinite value that all rows see: 57.8 us of a prompt of 1024 tokens, 36 without, 1284 of one of 8192, 567; 8 x 4
  // heads of 128.)
  for (bool careful = false;; careful = true) {
    bool large = false;  // some row's reference, times the scale
    ref = -INFINITY;
    base = sum = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; d++) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        acc[d][e] = 0.0f;
      }
    }
    for (int part = begin; part < end; part += kSteps) {
      int const part_end = end - part < kSteps ? end : part + kSteps;
      // Where the part's keys lie, in 16 bytes, and which of them exist, a bit each.  In the place of a key that does not any of the 64 that do: it is
      // masked, and what lies elsewhere may be no number.
      __syncthreads();
      for (int i = tid; i < (part_end - part + 63) / 64 * 64; i += kThreads) {
        int const key = part + i, real = key < kept ? key : key + shift, page = quotient(real, P.page_size, P.page_magic);
        int const number = key < part_end ? table[page] : -1;
        bool const is = (unsigned)number < (unsigned)P.pages;
        uint64_t const there = __ballot(is);
        uint32_t const step = (uint32_t)number * P.page_step + (uint32_t)(real - page * P.page_size) * P.token_step;
        uint32_t const some = there != 0 ? (uint32_t)__builtin_amdgcn_readlane((int)step, __builtin_ctzll(there)) : 0;
        steps[i] = is ? step : some;
        if (lane == 0) {
          exist[i / 64] = there;
        }
      }
      __syncthreads();

      // the rows that this thread loads chunks of, looked up a tile before their loads
      uint32_t from[LOADS];
      uint64_t there;
      auto locate = [&](int at) {
        int const in_part = at < part_end ? at - part : 0;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
          from[i] = steps[in_part + (kThreads * i + tid) / C] + chunk_of[i];
        }
        there = exist[in_part / 64];
      };
      auto load = [&](int buffer) {
        uint32_t const base = lds_at + buffer * 2 * tile_bytes<DP>() + 1024 * wave;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
          uint64_t const key = k_base + 16ull * from[i];
          paged::load_to_lds<false>(!padded || real[i] ? key : reinterpret_cast<uint64_t>(&paged::kZeros), base + 16 * kThreads * i);
        }
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
          paged::load_to_lds<false>(v_base + 16ull * from[i], base + tile_bytes<DP>() + 16 * kThreads * i);
        }
      };
      locate(part);
      load(0);
      uint64_t next_there = there;
      locate(part + KT);
      if (32 * __builtin_amdgcn_readfirstlane(wave) >= b.rows && !careful) {  // a wavefront without rows loads its share of the tiles, no more
        for (int at = part, buffer = 1; at < part_end; at += KT, buffer ^= 1) {
          paged::wait_loads<0>();
          __syncthreads();
          if (at + KT < part_end) {
            load(buffer);
          }
          locate(at + 2 * KT);
        }
        continue;
      }
      for (int at = part, buffer = 0; at < part_end; at += KT, buffer ^= 1) {
        uint64_t const is_there = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(next_there >> 32)) << 32 |
                                  (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)next_there);
        next_there = there;
        paged::wait_loads<0>();
        __syncthreads();  // the tile is here, and everyone is done with the one before
        if (at + KT < part_end) {
          load(buffer ^ 1);
        }
        unsigned char *const k_tile = lds + buffer * 2 * tile_bytes<DP>(), *const v_tile = k_tile + tile_bytes<DP>();

        floatx16 s[G];
#pragma unroll
        for (int j = 0; j < G; j++) {
#pragma unroll
          for (int e = 0; e < 16; e++) {
            s[j][e] = 0.0f;
          }
        }
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
#pragma unroll
          for (int j = 0; j < G; j++) {
            int const its = 32 * j + c;
            s[j] = mfma(*reinterpret_cast<x8 const *>(k_tile + its * (2 * DP) + 16 * place_of<C>(its, 2 * kk + h)), q[kk], s[j]);
          }
        }
        locate(at + 2 * KT);
        // operands of the products some ahead of them
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
        for (int i = 0; i < KK * G - 8; i++) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }

        // element e of s[j]: key 32 j + 8 (e / 4) + 4 h + e % 4 of row c
        int const half = KT == 32 ? (at - part) % 64 : 0;  // of a word of bits
        bool const all_there = KT == 64 ? is_there == ~0ull : (uint32_t)(is_there >> half) == ~0u;
        if (!all_there || __any(r.limit < at + KT || r.least > at) || careful) {
          uint32_t seen[G];
#pragma unroll
          for (int j = 0; j < G; j++) {
            int const first = at + 32 * j;
            seen[j] = (bits_below(r.limit - first) & ~bits_below(r.least - first)) | (TREE ? 0u : bits_below(r.always - first));
          }
          if constexpr (TREE) {
            int node = r.limit >= 0 ? r.token : -1;
            while (__any(node >= 0)) {
              int const place = context + node - at;
              if (node >= 0) {
#pragma unroll
                for (int j = 0; j < G; j++) {
                  seen[j] |= (unsigned)(place - 32 * j) < 32u ? 1u << (place - 32 * j) : 0u;
                }
                node = place > 0 ? tree[node] : -1;
              }
            }
          }
#pragma unroll
          for (int j = 0; j < G; j++) {
            seen[j] &= (uint32_t)(is_there >> (32 * j + half));
          }
          if (__builtin_expect(careful, 0)) {
            add_wild<T, DP>(v_tile, wild + 4, G == 1 ? seen[0] : (uint64_t)seen[G - 1] << 32 | seen[0], acc);
          }
#pragma unroll
          for (int j = 0; j < G; j++) {
            seen[j] >>= 4 * h;
#pragma unroll
            for (int e = 0; e < 16; e++) {
              s[j][e] = (seen[j] >> (8 * (e / 4) + e % 4)) & 1 ? s[j][e] : -INFINITY;
            }
          }
        }

        float top = s[0][0];
#pragma unroll
        for (int j = 0; j < G; j++) {
#pragma unroll
          for (int e = 0; e < 16; e++) {
            top = fmaxf(top, s[j][e]);
          }
        }
        top = over_halves(top, [](float a, float b) { return fmaxf(a, b); });
        if (__any((top - ref) * P.scale > kSlack) || large) {
          float const most = fmaxf(ref, top), from = most == -INFINITY ? 0.0f : most;
          float less = exp2_fast((ref - from) * P.scale);
          less = careful ? fmaxf(less, kNone) : less;
          ref = most;
          sum *= less;
#pragma unroll
          for (int d = 0; d < DB; d++) {
            acc[d] *= less;
          }
          large = __any(__builtin_fabsf(from) * P.scale > kLarge);
          base = most == -INFINITY ? 0.0f : (large ? bias : bias - from * P.scale);
          if (__builtin_expect(large, 0)) {
#pragma unroll
            for (int j = 0; j < G; j++) {
#pragma unroll
              for (int e = 0; e < 16; e++) {
                s[j][e] -= from;
              }
            }
          }
        }

        // Weights of sixteen keys at a time, and their products with the values.  O^T: lane has columns 32 d + 8 (e / 4) + 4 h + e % 4 of row c.
#pragma unroll
        for (int k = 0; k < 2 * G; k++) {
          x8 p;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            p[e] = static_cast<T>(exp2_fast(__builtin_fmaf(s[k / 2][8 * (k % 2) + e], P.scale, base)));
          }
          sum = sum_of(p, sum);
#pragma unroll
          for (int d = 0; d < DB; d++) {
            uint64_t v[2];
#pragma unroll
            for (int half = 0; half < 2; half++) {
              int const its = 16 * k + 8 * half + 4 * h + lane % 16 / 4, chunk = 4 * d + 2 * (lane / 16 % 2) + lane % 4 / 2;
              typedef short shortx4 __attribute__((ext_vector_type(4)));
              unsigned char const *const at_v = v_tile + its * (2 * DP) + 16 * place_of<C>(its, chunk) + 8 * (lane % 2);
              v[half] = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                         (shortx4 __attribute__((address_space(3))) *)(__attribute__((address_space(3))) void const *)at_v));
            }
            uintx4 const both = {(uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1], (uint32_t)(v[1] >> 32)};
            acc[d] = mfma(__builtin_bit_cast(x8, both), p, acc[d]);
          }
        }
      }
    }

    sum = over_halves(sum, [](float a, float b) { return a + b; });
    if (parts > 1 && 32 * wave < b.rows) {  // left as it is, for the kernel below
      int mine = tid;
      asm volatile("" : "+v"(mine));  // (places are not to be kept through the loop over tiles)
      int const wave = mine / 64, lane = mine % 64;
      float *const part = P.parts + (long long)blockIdx.x * part_floats<DP>();
      if (lane < 32) {
        part[kRows * DP + 2 * (32 * wave + lane)] = ref;
        part[kRows * DP + 2 * (32 * wave + lane) + 1] = sum;
      }
#pragma unroll
      for (int d = 0; d < DB; d++) {
#pragma unroll
        for (int four = 0; four < 4; four++) {
          *reinterpret_cast<paged::floatx4 *>(part + 4 * (((d * kWaves + wave) * 4 + four) * 64 + lane)) =
              paged::floatx4{acc[d][4 * four], acc[d][4 * four + 1], acc[d][4 * four + 2], acc[d][4 * four + 3]};
        }
      }
    }
    if (__builtin_expect(careful, 0)) {
      break;
    }
    // (columns past the head's end are its last ones again; without a sum of weights the row is NaN whatever the values are)
    paged::floatx4 none = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < DB; d++) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        none[e % 4] = __builtin_fmaf(acc[d][e], 0.0f, none[e % 4]);
      }
    }
    float const any = (none[0] + none[1]) + (none[2] + none[3]);
    bool const again = __any(any != any && sum == sum && is_row);
    if (lane == 0) {
      wild[wave] = again;
    }
    __syncthreads();
    if (__builtin_expect((wild[0] | wild[1] | wild[2] | wild[3]) == 0, 1)) {
      break;
    }
  }

  if (32 * wave >= b.rows || parts > 1) {
    return;
  }
  float const by = 1.0f / sum;
  int in_block = tid;
  asm volatile("" : "+v"(in_block));  // (the row's number and token are not to be kept through the loop over tiles)
  in_block = in_block / 64 * 32 + in_block % 32;
  int const row = b.row0 + (is_row ? in_block : 0), token = quotient(row, P.group, P.group_magic);
  T *const out = static_cast<T *>(P.out) + (long long)(b.row_of_q + token) * P.out_stride + (long long)(kv * P.group + row - token * P.group) * P.head_dim;
#pragma unroll
  for (int d = 0; d < DB; d++) {
#pragma unroll
    for (int four = 0; four < 4; four++) {
      x4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        y[e] = static_cast<T>(sum == 0.0f ? 0.0f : acc[d][4 * four + e] * by);
      }
      int const at = 32 * d + 8 * four + 4 * h;
      if (is_row && at < P.head_dim) {
        *reinterpret_cast<x4 *>(out + at) = y;
      }
    }
  }
}

// The parts of a block together, in the order in which the kernel above left them: WAYS wavefronts have 32 columns of 32 rows, each every
// WAYS-th part, asked for four at a time (one after the other each is a trip to memory), and then a share of the columns.
template <class T, int DP, bool TREE, int WAYS>
__global__ __launch_bounds__(kThreads) void join_blocks_kernel(BlockParams const P) {
  fetch_kernel_arguments<sizeof(BlockParams), 0>();
  constexpr int DB = DP / 32, kBatch = 4, kFours = 4 / WAYS;
  typedef typename Vec<T>::x4 x4;
  __shared__ paged::floatx4 shared_sums[WAYS][4][64];
  __shared__ float tops[WAYS][32], weights[WAYS][32];
  int const tid = threadIdx.x, lane = tid % 64, wave = tid / 64, way = wave % WAYS, h = lane / 32, c = lane % 32;
  int const d = (int)blockIdx.x % DB, rows = (int)blockIdx.x / DB % WAYS * kFours + wave / WAYS;
  int const kv = (int)blockIdx.x / (WAYS * DB) % P.kv_heads, block = (int)blockIdx.x / (WAYS * DB) / P.kv_heads;
  Block const b = block_of<TREE>(P, in_order<TREE>(P, block));
  if (!b.is || 32 * rows >= b.rows || 32 * d >= P.head_dim) {
    return;
  }
  int parts = parts_of(P, b), slot = block * P.kv_heads + kv, step = P.blocks * P.kv_heads;
  if (TREE && P.sequences > 1) {
    Cut const cut = cut_of<DP>(P, -1, b.sequence);
    parts = cut.parts;
    step = P.row_blocks * P.kv_heads;
    slot = cut.before + (block - b.sequence * P.row_blocks) * P.kv_heads + kv;
  }
  if (parts == 1) {
    return;  // (it has left the result)
  }
  int const in_block = 32 * rows + c;
  bool const is_row = in_block < b.rows;
  float top = -INFINITY, sum = 0.0f;
  paged::floatx4 x[4];
#pragma unroll
  for (int four = 0; four < 4; four++) {
    x[four] = paged::floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int i0 = way; i0 < parts; i0 += kBatch * WAYS) {
    float ref[kBatch], its[kBatch];
    paged::floatx4 y[kBatch][4];
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      int const which = i0 + i * WAYS < parts ? i0 + i * WAYS : i0;
      float const *const part = P.parts + (long long)(slot + which * step) * part_floats<DP>();
      ref[i] = part[kRows * DP + 2 * in_block];
      its[i] = part[kRows * DP + 2 * in_block + 1];
#pragma unroll
      for (int four = 0; four < 4; four++) {
        y[i][four] = *reinterpret_cast<paged::floatx4 const *>(part + 4 * (((d * kWaves + rows) * 4 + four) * 64 + lane));
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++) {  // (whether they count or not: what is asked for later is a trip of its own)
#pragma unroll
      for (int four = 0; four < 4; four++) {
        asm volatile("" : "+v"(y[i][four]));
      }
    }
    float const before = top;
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      ref[i] = i0 + i * WAYS < parts ? ref[i] : -INFINITY;
      top = fmaxf(top, ref[i]);
    }
    float const base = top == -INFINITY ? 0.0f : top, less = exp2_fast((before - base) * P.scale);
    sum *= less;
#pragma unroll
    for (int four = 0; four < 4; four++) {
      x[four] *= fmaxf(less, kNone);
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      float const by = exp2_fast((ref[i] - base) * P.scale);
      sum += its[i] * by;  // (NaN where every score is NaN that the row sees in the part, which then has no reference)
#pragma unroll
      for (int four = 0; four < 4; four++) {
        paged::floatx4 const z = fmaxf(by, kNone) * y[i][four];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[four][e] += i0 + i * WAYS < parts ? z[e] : 0.0f;
        }
      }
    }
  }
  if constexpr (WAYS > 1) {
    static_assert(WAYS == kWaves, "a workgroup is done with its rows, or joins them, as a whole");
#pragma unroll
    for (int four = 0; four < 4; four++) {
      shared_sums[way][four][lane] = x[four];
    }
    if (h == 0) {
      tops[way][c] = top;
      weights[way][c] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAYS; w++) {
      top = fmaxf(top, tops[w][c]);
    }
    float const base = top == -INFINITY ? 0.0f : top;
    sum = 0.0f;
    x[0] = paged::floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WAYS; w++) {
      float const by = exp2_fast((tops[w][c] - base) * P.scale);
      sum += weights[w][c] * by;
      x[0] += shared_sums[w][way][lane] * fmaxf(by, kNone);
    }
  }
  float const by = 1.0f / sum;
  int const row = b.row0 + (is_row ? in_block : 0), token = quotient(row, P.group, P.group_magic), d0 = 32 * d + 8 * way;
  T *const out = static_cast<T *>(P.out) + (long long)(b.row_of_q + token) * P.out_stride + (long long)(kv * P.group + row - token * P.group) * P.head_dim;
#pragma unroll
  for (int four = 0; four < kFours; four++) {
    int const at = d0 + 8 * four + 4 * h;
    if (is_row && at < P.head_dim) {
      x4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        y[e] = static_cast<T>(sum == 0.0f ? 0.0f : x[four][e] * by);
      }
      *reinterpret_cast<x4 *>(out + at) = y;
    }
  }
}

template <class T, int DP, bool TREE>
int launch_blocks(BlockParams P) {
  auto *fn = attention_blocks_kernel<T, DP, TREE>;
  constexpr int lds = lds_bytes<DP, TREE>();
  static_assert(kPerUnit<DP> * lds <= 160 * 1024, "LDS of a compute unit");
  P.row_blocks = (int)row_blocks((long long)P.new_tokens * P.group);
  P.blocks = (int)(P.starts == nullptr ? (long long)P.sequences * P.row_blocks : blocks_of(P.tokens, P.group, P.sequences));
  // Blocks that do not fill the chip are cut along their keys.
  long long const items = (long long)P.blocks * P.kv_heads, keys = (long long)P.table_width * P.page_size;
  long long const seen = P.window != 0 ? (long long)P.window + P.sinks + kRows : keys, most = seen < keys ? seen : keys;
  long long const room = (long long)(state().scratch_bytes / sizeof(float)) / part_floats<DP>(), fill = 256 * kPerUnit<DP>;
  P.slots = (int)(fill < room ? fill : room);
  long long splits = P.slots / items;
  // Parts of a tile where that gives no more than one for each compute unit and sixteen to be joined (a trip to memory), of two otherwise.  Measured
  // (us, two and one; 8 heads of 128, 48 rows): 14.8 and 14.0 of one sequence of 1000 keys, 13.2 and 11.5 of 300; against it 15.1 and 16.8 of one of 2000,
  // 17.8 and 19.4 of three of up to 1000, 96 rows.
  P.least = most <= 1024 && items * ((most + 63) / 64) <= 256 ? 64 : 128;
  splits = splits < most / P.least ? splits : most / P.least;
  splits = splits < room / items ? splits : room / items;
  P.splits = splits < 1 ? 1 : (int)splits;
  // Trees behind contexts of different lengths are cut where that evens out what workgroups have to do, joins included.  Measured (us, whole and cut;
  // 8 heads of 128): 126 and 92 of 36 trees behind up to 4096 keys, 145 and 131 of 48, 63 and 53 of 36 behind up to 2000; against it 75 and 85 of 64 behind
  // up to 2000, 22.7 and 29.2 of 48 behind up to 400.
  if (TREE && P.sequences > 1 && P.splits == 1 && items * 5 <= P.slots * 4 && keys >= 1536) {
    P.splits = 2;
  }
  P.parts = static_cast<float *>(state().scratch());
  MI355_GRANT_LDS(fn, lds);
  long long const grid = TREE && P.sequences > 1 && P.splits > 1 ? P.slots : items * P.splits;
  MI355_HIP(launch_kernel(fn, dim3((unsigned)grid), dim3(kThreads), lds, state().stream(), P));
  if (P.splits > 1) {
    // Four wavefronts to the parts of the same rows where there are many parts of few rows: 19.4 and 22.8 us with and without of 5 x 3 heads of 80 x up to
    // 3001 keys, 65 rows, 14.9 and 15.6 of 1 x 8 of 128 x 1000, 48 rows; against it 37.9 and 35.4 of 12 x 8 of 128 x up to 4096, 96 rows.
    bool const several = P.splits > 4 && items * (DP / 8) <= 1024;
    auto *join = several ? join_blocks_kernel<T, DP, TREE, 4> : join_blocks_kernel<T, DP, TREE, 1>;
    MI355_HIP(launch_kernel(join, dim3((unsigned)(items * (DP / (several ? 8 : 32)))), dim3(kThreads), 0, state().stream(), P));
  }
  return MI355_OK;
}

template <class T, bool TREE>
int launch_head(BlockParams const &P) {
  return P.head_dim <= 64    ? launch_blocks<T, 64, TREE>(P)
         : P.head_dim <= 96  ? launch_blocks<T, 96, TREE>(P)
         : P.head_dim <= 128 ? launch_blocks<T, 128, TREE>(P)
         : P.head_dim <= 192 ? launch_blocks<T, 192, TREE>(P)
                             : launch_blocks<T, 256, TREE>(P);
}

}  // namespace blocks
}  // namespace mi355
