// Attention of blocks of rows over a paged key-value cache: whole prompts and chunks of them within a window, and trees of
// drafted tokens.
//
// o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q . k_j, over the keys a row sees, in one pass with a running
// maximum.  A row is a new token and one of the query heads that share a key-value head, so that these heads share its keys too.
// * A workgroup has 128 rows, a wavefront 32 of them; tiles of keys and values come from the pages straight into LDS, the next
//   while one is worked on: one barrier a tile.
// * Scores are made transposed, S^T = K Q^T, by products of 32 x 32 x 16: a lane then has half the weights of one row, of the
//   keys that it has as the operand of O^T = V^T P^T if values are read in that order.  No weight changes lanes.
// * Keys are counted as the block sees them: the first `kept` of the sequence, then those from `first` on, in one run without a gap
//   (a tile has 64 lanes to look up a key each, so a run may jump anywhere).
// * Weights are rounded to the values' type once: as much error again as rounding the result makes, at two thirds of the matrix
//   products that exact ones would take.
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

// Where 16-byte chunk `chunk` of row `row` lies in a tile of C chunks a row (64 banks of 4 bytes: sixteen chunks).  Sixteen rows read
// the same chunk of K; four rows read four chunks of V in a row.
template <int C, bool VALUES>
__device__ __forceinline__ int turn_of(int row) {
  return VALUES ? (C == 8 || C == 24 ? 4 * ((row >> 1) & 1) : C == 12 ? 0 : 4 * (row & 3))
                : (C == 8 || C == 24 ? (row >> 1) & 7 : C == 12 ? (row >> 2) & 3 : row & 15);
}
template <int C, bool VALUES>
__device__ __forceinline__ int place_of(int row, int chunk) {
  int const turn = turn_of<C, VALUES>(row);
  if constexpr ((C & (C - 1)) == 0) {
    return chunk ^ turn;
  }
  int const at = chunk + turn;
  return at >= C ? at - C : at;
}
template <int C, bool VALUES>
__device__ __forceinline__ int chunk_at(int row, int place) {
  int const turn = turn_of<C, VALUES>(row);
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

__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1); }

constexpr int kThreads = 256, kWaves = 4, kIds = 1024;
template <int DP>
constexpr int kKeys = DP <= 128 ? 64 : 32;  // of a tile
template <int DP>
constexpr int tile_bytes() { return kKeys<DP> * DP * 2; }
template <int DP, bool TREE>
constexpr int lds_bytes() { return 4 * tile_bytes<DP>() + 4 * kIds + (TREE ? 4 * MI355_MAX_TREE_NODES : 0); }

template <class T, int DP, bool TREE>
__global__ __launch_bounds__(kThreads, 2) void attention_blocks_kernel(BlockParams const P) {
  fetch_kernel_arguments<sizeof(BlockParams), 1>();
  constexpr int KT = kKeys<DP>, G = KT / 32, C = DP / 8, LOADS = KT * C / kThreads, KK = DP / 16, DB = DP / 32;
  typedef typename Vec<T>::x8 x8;
  typedef typename Vec<T>::x4 x4;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  int *const ids = reinterpret_cast<int *>(lds + 4 * tile_bytes<DP>());
  int *const tree = ids + kIds;
  int const tid = threadIdx.x, lane = tid % 64, wave = tid / 64, h = lane / 32, c = lane % 32;
  uint32_t const lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void const *)lds;

  // the block: key-value heads side by side (eight of them lie on an XCD each, with the keys that its blocks share)
  int const kv = (int)blockIdx.x % P.kv_heads;
  int block = (int)blockIdx.x / P.kv_heads, sequence = 0, row_of_q = 0, new_tokens = P.new_tokens;
  if (P.starts == nullptr) {
    sequence = block / P.row_blocks;
    block -= sequence * P.row_blocks;
    row_of_q = sequence * P.new_tokens;
  } else {
    for (int base = 0;; base += 64) {
      if (base >= P.sequences) {
        return;
      }
      int const b = base + lane;
      auto start = [&](int i) {
        int const s = P.starts[i];
        return s < 0 ? 0 : (s < P.tokens ? s : P.tokens);
      };
      int const from = b < P.sequences ? start(b) : 0, to = b < P.sequences ? start(b + 1) : 0;
      int const its = to > from ? (int)(((long long)(to - from) * P.group + kRows - 1) / kRows) : 0, upto = paged::wave_upto(its);
      uint64_t const past = __ballot(upto > block);
      if (past != 0) {
        int const at = __builtin_ctzll(past);
        sequence = base + at;
        row_of_q = __builtin_amdgcn_readlane(from, at);
        new_tokens = __builtin_amdgcn_readlane(to, at) - row_of_q;
        block -= __builtin_amdgcn_readlane(upto - its, at);
        break;
      }
      block -= __builtin_amdgcn_readlane(upto, 63);
    }
  }

  // its rows and the keys that any of them sees, counted as kept + those from `first` on
  int const R = new_tokens * P.group, row0 = block * kRows, rows = R - row0 < kRows ? R - row0 : kRows;
  int const most = P.table_width * P.page_size, told = P.lengths[sequence];
  int const length = told < 0 ? 0 : (told < most ? told : most);
  auto token_of = [&](int row) { return quotient(row, P.group, P.group_magic); };
  auto limit_of = [&](int t) { return length - (new_tokens - 1 - t); };
  int const context = length - new_tokens;  // of a tree
  int to = TREE ? length : limit_of(token_of(row0 + rows - 1));
  to = to < 0 ? 0 : to;
  int first = !TREE && P.window != 0 ? limit_of(token_of(row0)) - P.window : 0;
  first = first < 0 ? 0 : first;
  int const kept = P.sinks < first ? P.sinks : first, shift = first - kept, end = to - shift;

  // this lane's row: the run's keys below `always`, and those from `least` up to `limit`
  int const row = row0 + 32 * wave + c, my_token = token_of(row < R ? row : R - 1);
  int limit = 0, least = 0, always = 0;
  if (row < R) {
    limit = TREE ? context : limit_of(my_token) - shift;
    least = !TREE && P.window != 0 ? limit - P.window : 0;
    always = P.sinks < limit ? P.sinks : limit;
  }

  x8 q[KK];
  {
    T const *const from = static_cast<T const *>(P.q) + (long long)(row_of_q + my_token) * P.q_stride +
                          (long long)(kv * P.group + (row < R ? row : R - 1) - my_token * P.group) * P.head_dim;
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
      int const d = 16 * kk + 8 * h;
      uintx4 x = {0, 0, 0, 0};
      if (row < R && d < P.head_dim) {
        x = *reinterpret_cast<uintx4 const *>(from + d);
      }
#pragma unroll
      for (int w = 0; w < 4; w++) {
        x[w] = (x[w] & P.q_keep) ^ P.q_flip;
      }
      q[kk] = __builtin_bit_cast(x8, x);
    }
  }
  if constexpr (TREE) {
    for (int i = tid; i < new_tokens; i += kThreads) {
      tree[i] = P.parents[(long long)sequence * new_tokens + i];
    }
    __syncthreads();
    // whether every ancestor is there: else the row sees nothing
    int at = row < R && context + my_token >= 0 ? my_token : -2;
    while (__any(at >= 0)) {
      if (at >= 0) {
        int const p = tree[at];
        at = p >= -1 && p < at && (p < 0 || context + p >= 0) ? p : -2;
      }
    }
    limit = at == -1 ? (limit < 0 ? 0 : limit) : -1;
  }

  floatx16 acc[DB];
  float ref = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < DB; d++) {
#pragma unroll
    for (int e = 0; e < 16; e++) {
      acc[d][e] = 0.0f;
    }
  }
  // Weights are at most 2^(bias + kSlack): the reference follows the maximum only where that would be passed, so that sums are seldom
  // scaled.  fp16: small ones stay above the type's end.  bf16: as values reach the end of 32 bits themselves, n weights add up to less than 1/2.
  constexpr float kSlack = 6.0f;
  float const bias = std::is_same<T, _Float16>::value ? 9.0f : (float)(__builtin_clz((unsigned)end | 1u) - 33) - kSlack;
  uint64_t const k_base = reinterpret_cast<uint64_t>(P.k) + 16ull * kv * P.head_step, v_base = reinterpret_cast<uint64_t>(P.v) + 16ull * kv * P.head_step;
  int const *const table = P.table + (long long)sequence * P.table_width;

  // as many keys at a time as the page numbers in LDS cover
  int const fit = P.page_size < 1 << 16 ? (kIds - 4) * P.page_size / KT * KT : 1 << 25;
  for (int part = 0; part < end; part += fit) {
    int const part_end = end - part < fit ? end : part + fit;
    auto page_of = [&](int key) { return quotient(key, P.page_size, P.page_magic); };
    int const kept_page = page_of(part), kept_end = part_end < kept ? part_end : kept;
    int const kept_pages = part < kept ? page_of(kept_end - 1) + 1 - kept_page : 0;
    int const later = part > kept ? part : kept, later_page = later < part_end ? page_of(later + shift) : 0;
    int const later_pages = later < part_end ? page_of(part_end - 1 + shift) + 1 - later_page : 0;
    __syncthreads();
    for (int i = tid; i < kept_pages + later_pages; i += kThreads) {
      ids[i] = table[i < kept_pages ? kept_page + i : later_page + i - kept_pages];
    }
    __syncthreads();

    uint64_t there = 0;  // keys of the tile that exist, a bit each
    auto load = [&](int at, int buffer) {
      int const key = at + lane % KT, real = key < kept ? key : key + shift, page = page_of(real);
      int const number = key < part_end ? ids[key < kept ? page - kept_page : kept_pages + page - later_page] : -1;
      bool const is = (unsigned)number < (unsigned)P.pages;
      there = __ballot(is);
      uint32_t const step = is ? (uint32_t)number * P.page_step + (uint32_t)(real - page * P.page_size) * P.token_step : ~0u;
      int chunks = P.head_dim / 8;
      asm volatile("" : "+s"(chunks));
      uint32_t const base = lds_at + buffer * 2 * tile_bytes<DP>() + 1024 * wave;
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        int const n = kThreads * i + tid, its = n / C, k_chunk = chunk_at<C, false>(its, n % C), v_chunk = chunk_at<C, true>(its, n % C);
        uint32_t const from = (uint32_t)__shfl((int)step, its, 64);
        uint64_t const zeros = reinterpret_cast<uint64_t>(&paged::kZeros);
        paged::load_to_lds<false>(from != ~0u && k_chunk < chunks ? k_base + 16ull * (from + k_chunk) : zeros, base + 16 * kThreads * i);
        paged::load_to_lds<false>(from != ~0u && v_chunk < chunks ? v_base + 16ull * (from + v_chunk) : zeros,
                                  base + tile_bytes<DP>() + 16 * kThreads * i);
      }
    };
    load(part, 0);
    for (int at = part, buffer = 0; at < part_end; at += KT, buffer ^= 1) {
      uint64_t const is_there = there;
      paged::wait_loads<0>();
      __syncthreads();  // the tile is here, and everyone is done with the one before
      if (at + KT < part_end) {
        load(at + KT, buffer ^ 1);
      }
      unsigned char const *const k_tile = lds + buffer * 2 * tile_bytes<DP>(), *const v_tile = k_tile + tile_bytes<DP>();

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
          s[j] = mfma(*reinterpret_cast<x8 const *>(k_tile + its * (2 * DP) + 16 * place_of<C, false>(its, 2 * kk + h)), q[kk], s[j]);
        }
      }

      // element e of s[j]: key 32 j + 8 (e / 4) + 4 h + e % 4 of row c
      bool const all_there = is_there == (KT == 64 ? ~0ull : 0xffffffffull);
      if (!all_there || __any(limit < at + KT || least > at)) {
        uint32_t seen[G];
#pragma unroll
        for (int j = 0; j < G; j++) {
          int const from = at + 32 * j;
          seen[j] = (bits_below(limit - from) & ~bits_below(least - from)) | (TREE ? 0u : bits_below(always - from));
        }
        if constexpr (TREE) {
          int node = limit >= 0 ? my_token : -1;
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
          seen[j] = (seen[j] & (uint32_t)(is_there >> (32 * j))) >> (4 * h);
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
      top = over_halves(top, [](float a, float b) { return fmaxf(a, b); }) * P.scale;
      if (__any(top > ref + kSlack || (ref == -INFINITY && top > ref))) {
        float const higher = fmaxf(ref, top), less = exp2_fast(ref - (higher == -INFINITY ? 0.0f : higher));
        ref = higher;
        sum *= less;
#pragma unroll
        for (int d = 0; d < DB; d++) {
          acc[d] *= less;
        }
      }
      float const base = ref == -INFINITY ? 0.0f : bias - ref;
      x8 p[2 * G];
#pragma unroll
      for (int j = 0; j < G; j++) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
          float const w = exp2_fast(__builtin_fmaf(s[j][e], P.scale, base));
          sum += w;
          p[2 * j + e / 8][e % 8] = static_cast<T>(w);
        }
      }

      // O^T: lane has columns 32 d + 8 (e / 4) + 4 h + e % 4 of row c
#pragma unroll
      for (int k = 0; k < 2 * G; k++) {
#pragma unroll
        for (int d = 0; d < DB; d++) {
          uint64_t v[2];
#pragma unroll
          for (int half = 0; half < 2; half++) {
            int const its = 16 * k + 8 * half + 4 * h + lane % 16 / 4, chunk = 4 * d + 2 * (lane / 16 % 2) + lane % 4 / 2;
            typedef short shortx4 __attribute__((ext_vector_type(4)));
            unsigned char const *const from = v_tile + its * (2 * DP) + 16 * place_of<C, true>(its, chunk) + 8 * (lane % 2);
            v[half] = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                       (shortx4 __attribute__((address_space(3))) *)(__attribute__((address_space(3))) void const *)from));
          }
          uintx4 const both = {(uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1], (uint32_t)(v[1] >> 32)};
          acc[d] = mfma(__builtin_bit_cast(x8, both), p[k], acc[d]);
        }
      }
    }
  }

  sum = over_halves(sum, [](float a, float b) { return a + b; });
  float const by = sum == 0.0f ? 0.0f : 1.0f / sum;
  bool good = true;
  T *const out = static_cast<T *>(P.out) + (long long)(row_of_q + my_token) * P.out_stride + (long long)(kv * P.group + row - my_token * P.group) * P.head_dim;
#pragma unroll
  for (int d = 0; d < DB; d++) {
#pragma unroll
    for (int four = 0; four < 4; four++) {
      x4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float const o = acc[d][4 * four + e] * by;
        good = good && __builtin_fabsf(o) < INFINITY;  // (false for NaN)
        y[e] = static_cast<T>(o);
      }
      int const at = 32 * d + 8 * four + 4 * h;
      if (row < R && at < P.head_dim) {
        *reinterpret_cast<x4 *>(out + at) = y;
      }
    }
  }

  // A weight of zero does not keep an infinity or NaN among the values out of a sum: rows with one in their result are done again,
  // a wavefront a row, key by key.  (In the loop above such values would have to be looked for in every tile that not all rows see.)
  uint64_t again = __ballot(!good && row < R);
  again = (again | again >> 32) & 0xffffffffull;
  for (; again != 0; again &= again - 1) {
    int const which = __builtin_ctzll(again), its_row = row0 + 32 * wave + which, t = token_of(its_row);
    int const its_limit = __builtin_amdgcn_readlane(limit, which), its_least = __builtin_amdgcn_readlane(least, which);
    int const its_always = __builtin_amdgcn_readlane(always, which);
    T const *const its_q = static_cast<T const *>(P.q) + (long long)(row_of_q + t) * P.q_stride + (long long)(kv * P.group + its_row - t * P.group) * P.head_dim;
    T *const its_out = static_cast<T *>(P.out) + (long long)(row_of_q + t) * P.out_stride + (long long)(kv * P.group + its_row - t * P.group) * P.head_dim;
    bool const negative = P.q_flip != 0, none = P.q_keep == 0;
    // the key of this lane of 64: where it lies, or all ones where the row does not see it
    auto find = [&](int key) {
      int const real = key < kept ? key : key + shift, page = quotient(real, P.page_size, P.page_magic);
      bool sees = key < end && ((key < its_limit && key >= its_least) || (!TREE && key < its_always));
      if constexpr (TREE) {
        if (its_limit >= 0) {
          for (int node = t; node >= 0; node = tree[node]) {
            sees = sees || key == context + node;
          }
        }
      }
      int const number = sees ? table[page] : -1;
      return (unsigned)number < (unsigned)P.pages ? (uint32_t)number * P.page_step + (uint32_t)(real - page * P.page_size) * P.token_step : ~0u;
    };
    auto score = [&](uint32_t at) {
      float x = 0.0f;
      if (at == ~0u) {
        return -INFINITY;
      }
      for (int d = 0; d < P.head_dim; d += 8) {
        x8 const k = *reinterpret_cast<x8 const *>(k_base + 16ull * (at + d / 8)), a = *reinterpret_cast<x8 const *>(its_q + d);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          x += static_cast<float>(a[e]) * static_cast<float>(k[e]);
        }
      }
      x = none ? x * 0.0f : x;
      return (negative ? -x : x) * P.scale;
    };
    float high = -INFINITY;
    bool wild = false;
    for (int key = 0; key < end; key += 64) {
      float const x = score(find(key + lane));
      wild = wild || x != x;
      high = fmaxf(high, x);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      high = fmaxf(high, __shfl_xor(high, off, 64));
    }
    wild = __any(wild) || high == INFINITY;
    float total = 0.0f, o[DP / 64 + 1];
#pragma unroll
    for (int i = 0; i <= DP / 64; i++) {
      o[i] = 0.0f;
    }
    float const from_high = high == -INFINITY ? 0.0f : bias - high;
    for (int key = 0; key < end && !wild; key += 64) {
      uint32_t const at = find(key + lane);
      float const w = at == ~0u ? 0.0f : exp2_fast(score(at) + from_high);
      total += w;
      for (uint64_t left = __ballot(at != ~0u); left != 0; left &= left - 1) {
        int const j = __builtin_ctzll(left);
        float const its = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j));
        T const *const v = reinterpret_cast<T const *>(v_base + 16ull * (uint32_t)__builtin_amdgcn_readlane((int)at, j));
#pragma unroll
        for (int i = 0; i <= DP / 64; i++) {
          if (64 * i + lane < P.head_dim) {
            float const x = static_cast<float>(v[64 * i + lane]);
            o[i] += __builtin_fabsf(x) == INFINITY && high != -INFINITY ? x : its * x;
          }
        }
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      total += __shfl_xor(total, off, 64);
    }
#pragma unroll
    for (int i = 0; i <= DP / 64; i++) {
      if (64 * i + lane < P.head_dim) {
        its_out[64 * i + lane] = static_cast<T>(wild ? __builtin_nanf("") : (total == 0.0f ? 0.0f : o[i] * (1.0f / total)));
      }
    }
  }
}

template <class T, int DP, bool TREE>
int launch_blocks(BlockParams const &P) {
  auto *fn = attention_blocks_kernel<T, DP, TREE>;
  constexpr int lds = lds_bytes<DP, TREE>();
  static_assert(2 * lds <= 160 * 1024, "two workgroups to a compute unit");
  long long const blocks = P.starts == nullptr ? (long long)P.sequences * P.row_blocks : blocks_of(P.tokens, P.group, P.sequences);
  MI355_GRANT_LDS(fn, lds);
  MI355_HIP(launch_kernel(fn, dim3((unsigned)(blocks * P.kv_heads)), dim3(kThreads), lds, state().stream(), P));
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
