// Attention of a sequence's new tokens over a paged key-value cache.
//
// o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q . k_j, over the keys a row sees, in one pass with the
// running maximum m: when it grows, what has been summed is scaled down.
//
// Every key and value is read once for all rows of its head (query heads of the group x new tokens), so the bytes of
// the cache bound a long call and the chain of trips to memory a short one.  What follows from that:
// * the work is cut into units of 32, 128 or 256 keys (32 a wavefront, of which a workgroup has one, four or eight) of one sequence and
//   key-value head.  Every head goes in equal parts to as many workgroups as its share of the chip is, or, where heads are more or
//   shorter than that, units are dealt in equal runs that go on from one head to the next.  The parts of a head are joined
//   by the last of its workgroups (a ticket), in the order of the keys; more than eight in levels.
// * a wavefront has 32 keys at a time and streams them from the pages straight into LDS of its own: no barrier in the
//   loop.  The next keys are on their way while the scores become weights, the next values while the next scores are made.
//   Waits count the transfers of the younger tile; anything else in flight would only make them wait for more.
// * scores are made transposed, S^T = K Q^T: a lane then has the weights of one row, as the operand of O^T = V^T P^T
//   wants them, and that row's maximum, sum and scale.
#pragma once

#include "common.h"
#include "mi355_kernels/kernarg.h"
#include "mi355_kernels/paged_units.h"

#include <climits>
#include <cmath>
#include <type_traits>

namespace mi355 {
namespace paged {

template <int WAVES>
constexpr int kIdsOf = WAVES == 1 ? 256 : 1024;  // page numbers of a run that a workgroup holds in LDS
constexpr int kAtOnce = 8;                // parts that a thread reads together; more are joined in levels

struct PagedParams {
  void const *q, *k, *v;
  void *out;
  long long q_stride, out_stride;
  uint32_t page_step, token_step, head_step;  // in 16 bytes: a cache is up to 64 GB
  int const *table, *lengths;
  float *parts;   // 2 per workgroup: the end of a head that began before it, the beginning of one that goes on after it
  int *tickets;   // kTicketsEach per workgroup, kJoinStep apart, zero between launches
  int pages, page_size, head_dim, table_width, sequences, new_tokens, group, window;
  int row_blocks, heads;  // of 16 RG rows, of a key-value head; key-value heads x row blocks
  unsigned page_magic, group_magic;  // see quotient
  uint32_t q_keep, q_flip;           // bits of queries: a scale of zero or below zero is in them
  float scale;                       // its magnitude, times log2 e: weights are powers of two
};

// n / d for 0 <= n < 2^31 - d by magic = 2^32 / d, rounded up (0 for d = 1): one too many at most
__device__ __forceinline__ int quotient(int n, int d, unsigned magic) {
  int const q = magic == 0 ? n : (int)__umulhi((uint32_t)n, magic);
  return q - (q * d > n ? 1 : 0);
}
inline unsigned magic_of(int d) { return d == 1 ? 0 : (unsigned)(((1ull << 32) + d - 1) / d); }

// The two units of this operator: the kernels of a type are compiled in one of them each, side by side.
int launch_f16(PagedParams const &P, int kv_heads, bool passing);
int launch_bf16(PagedParams const &P, int kv_heads, bool passing);

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
template <class T>
struct Vec {
  typedef T x8 __attribute__((ext_vector_type(8)));
  typedef T x4 __attribute__((ext_vector_type(4)));
  static constexpr uint32_t exponent = sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7c00 : 0x7f80;  // all ones: no number
};

__device__ __forceinline__ floatx4 mfma(Vec<_Float16>::x8 a, Vec<_Float16>::x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mfma(Vec<__bf16>::x8 a, Vec<__bf16>::x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// What a masked key and the columns past a head's end are loaded from.
static __device__ uintx4 const kZeros = {0, 0, 0, 0};

// Every lane fetches 16 bytes from an address of its own; they land at `lds` + 16 * lane (vmcnt counts the transfer; the
// caller waits).  Inline assembly because the compiler would have the next LDS read of any address wait for all of them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <bool PASSING>  // PASSING: not to be kept in the caches
__device__ __forceinline__ void load_to_lds(uint64_t address, uint32_t lds) {
  if constexpr (PASSING) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(address)
                 : "m0", "memory");
  } else {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(address)
                 : "m0", "memory");
  }
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// Where 16-byte chunk `chunk` of row `row` of a tile lies in it, and what lies where.  The sixteen rows of a score
// operand read the same chunk of K, the eight of half a transposing read the same pair of V: their places are turned by
// the row so that they fall on different banks (64 of 4 bytes: sixteen chunks in a row).  C chunks a row.
template <int C, bool VALUES>
__device__ __forceinline__ int turn_of(int row) {
  return VALUES ? (C == 8 ? 2 * ((row >> 1) & 3) : C == 12 ? 2 * ((row >> 2) & 1) : C == 24 ? 2 * ((row >> 1) & 3) : 2 * (row & 7))
                : (C == 8 ? (row >> 1) & 7 : C == 12 ? (row >> 2) & 3 : C == 24 ? (row >> 1) & 7 : row & 15);
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

// x[l] op x[l ^ 16] op x[l ^ 32] op x[l ^ 48] in every lane: over the four groups of lanes that share a row.  By the
// instructions that exchange rows of 16 lanes and halves of a wavefront between two registers; a shuffle is a trip through
// LDS.  (Inline assembly: the compiler's builtin returns the first result twice.  The wait states cover a write just before.)
template <class Op>
__device__ __forceinline__ float over_groups(float x, Op op) {
  float a = x, b = x;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  a = b = op(a, b);
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return op(a, b);
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Two weights as two numbers of the value's type each, of which the second is what cutting the first short lost and a small
// part of the first beside it, so that it is not zero: zero times an infinite value would be NaN where the sum is infinite.
// All weights grow by that part alike (divided out at the end) but for what is cut off, a 2^-10 (2^-7) of one at most.
template <class T>
constexpr float kPart = std::is_same<T, _Float16>::value ? 0x1p-8f : 0x1p-12f;
__device__ __forceinline__ void split(float w0, float w1, uint32_t &first, uint32_t &rest, _Float16) {
  constexpr float back = kPart<_Float16> - 1.0f;
  auto const cut = __builtin_amdgcn_cvt_pkrtz(w0, w1);
  auto const less = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf(back, static_cast<float>(cut[0]), w0), __builtin_fmaf(back, static_cast<float>(cut[1]), w1));
  first = __builtin_bit_cast(uint32_t, cut);
  rest = __builtin_bit_cast(uint32_t, less);
}
__device__ __forceinline__ void split(float w0, float w1, uint32_t &first, uint32_t &rest, __bf16) {
  constexpr float back = kPart<__bf16> - 1.0f;
  uint32_t const b0 = __builtin_bit_cast(uint32_t, w0), b1 = __builtin_bit_cast(uint32_t, w1);
  first = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  pair const less = {static_cast<__bf16>(__builtin_fmaf(back, __builtin_bit_cast(float, b0 & 0xffff0000u), w0)),
                     static_cast<__bf16>(__builtin_fmaf(back, __builtin_bit_cast(float, b1 & 0xffff0000u), w1))};
  rest = __builtin_bit_cast(uint32_t, less);
}

struct Span {
  int first, to;  // the keys that any row sees
  int from;       // the tile that the first of them lies in
  int units;     // at least one: a head without keys has its zeros to be written
};
template <int UNIT>
__device__ __forceinline__ Span span_of(PagedParams const &P, int told) {  // of the sequence with that length
  int const most = P.table_width * P.page_size;
  int const length = told < 0 ? 0 : (told < most ? told : most);
  int const first = P.window != 0 ? length - (P.new_tokens - 1) - P.window : 0;  // (no underflow: the host bounds both)
  Span s;
  s.first = first > 0 ? first : 0;
  s.from = s.first & ~(kTile - 1);
  s.to = length;
  s.units = length > s.from ? (length - s.from + UNIT - 1) / UNIT : 1;
  return s;
}

// the sum of the lanes up to this one, by moves between registers: within rows of 16, then the ends of rows
__device__ __forceinline__ int wave_upto(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // from 1, 2, 4, 8 lanes before in the row
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true);  // the end of rows 0 and 2 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true);  // the end of row 1 to rows 2 and 3
  return x;
}

// Parts go through the memory that all XCDs share: device-scope stores and loads (sc1 on each), which pass by this XCD's L2.
// The join depends on that for every access to a part, not on fences: parts lie where those of earlier launches did, and
// a load that this XCD's L2 may serve finds what was there then.  The ticket is taken when the stores have arrived (vmcnt).
__device__ __forceinline__ void store_shared(float *p, float a, float b) {
  uint64_t const both = (uint64_t)__builtin_bit_cast(uint32_t, a) | (uint64_t)__builtin_bit_cast(uint32_t, b) << 32;
  __hip_atomic_store((__attribute__((address_space(1))) uint64_t *)(uint64_t *)p, both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_shared(float *p, floatx4 v) {
  store_shared(p, v[0], v[1]);
  store_shared(p + 2, v[2], v[3]);
}
__device__ __forceinline__ uint64_t load_shared(float const *p) {
  return __hip_atomic_load((__attribute__((address_space(1))) uint64_t const *)(uint64_t const *)p, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float low_of(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)x); }
__device__ __forceinline__ float high_of(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)(x >> 32)); }

template <int DP, int RG>
constexpr int part_floats() { return 16 * RG * (DP + 4); }  // rows of numerators, then each one's maximum and sum, twice
template <int DP>
constexpr int tile_bytes() { return kTile * DP * 2; }
template <int DP, int RG>
constexpr int query_bytes() { return RG > 1 ? 16 * RG * DP * 2 : 0; }
// tiles, and queries where they are too many for registers; at a head's end in their place the wavefronts' sums, whose rows
// begin at other banks than their neighbours (a lane of each writes at once: a row after the other took 1 us)
template <int DP>
constexpr int sum_row() { return DP + 4; }
template <int DP, int RG, int WAVES>
constexpr int tiles_bytes() {
  constexpr int tiles = WAVES * 2 * tile_bytes<DP>() + query_bytes<DP, RG>(), sums = WAVES * 16 * RG * sum_row<DP>() * 4;
  return tiles > sums ? tiles : sums;
}
// behind them page numbers; maximum and sum of every wavefront's rows; what a row is to be multiplied by; whether this workgroup
// is the last
template <int DP, int RG, int WAVES>
constexpr int lds_bytes() { return tiles_bytes<DP, RG, WAVES>() + (int)sizeof(int) * kIdsOf<WAVES> + WAVES * 16 * RG * 8 + 16 * RG * 4 + 16; }

// Workgroups that a compute unit's LDS and registers hold.
template <int DP, int RG, int WAVES>
constexpr int per_compute_unit() {
  constexpr int by_lds = 160 * 1024 / lds_bytes<DP, RG, WAVES>(), by_registers = (DP <= 128 && RG < 4 && RG * DP <= 288 ? 8 : 4) / WAVES;
  return WAVES == 8 ? 1 : (by_lds < by_registers ? by_lds : by_registers);
}

// DP: the head size, rounded up; RG: groups of 16 rows; WAVES: wavefronts of a workgroup; PASSING: keys and values are not to
// be kept in the caches.
template <class T, int DP, int RG, int WAVES, bool PASSING>
__global__ __launch_bounds__(64 * WAVES, ((WAVES * per_compute_unit<DP, RG, WAVES>() + 3) / 4)) void paged_attention_kernel(PagedParams const P) {
  fetch_kernel_arguments<sizeof(PagedParams), 1>();  // one trip for all of them
  constexpr int kWaves = WAVES, kThreads = 64 * WAVES, kUnit = kTile * WAVES, kIds = kIdsOf<WAVES>;
  constexpr int C = DP / 8, LOADS = kTile * C / 64, KK = DP / 32, DB = DP / 16;
  typedef typename Vec<T>::x8 x8;
  typedef typename Vec<T>::x4 x4;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  unsigned char *const queries = lds + kWaves * 2 * tile_bytes<DP>();
  int *const ids = reinterpret_cast<int *>(lds + tiles_bytes<DP, RG, WAVES>());
  float *const stat = reinterpret_cast<float *>(ids + kIds);
  float *const row_by = stat + kWaves * 16 * RG * 2;
  int *const is_last = reinterpret_cast<int *>(row_by + 16 * RG);
  int const tid = threadIdx.x, lane = tid % 64, wave = tid / 64, g = lane / 16, c = lane % 16;
  unsigned char *const k_tile = lds + wave * 2 * tile_bytes<DP>(), *const v_tile = k_tile + tile_bytes<DP>();
  uint32_t const k_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void const *)k_tile;
  uint32_t const v_lds = k_lds + tile_bytes<DP>();

  // This workgroup's units.  Every head cut into equal parts of at most `run` units, a workgroup each, where that gives
  // no more parts than workgroups; otherwise (heads shorter than a run) runs of units that go on from one head to the next.
  int const own_length = lane < P.sequences ? P.lengths[lane] : 0;
  int const own_units = lane < P.sequences ? span_of<kUnit>(P, own_length).units : 0;
  auto over_sequences = [&](auto value) {  // the sum of value(units of a sequence)
    int x = lane < P.sequences ? value(own_units) : 0;
    for (int b = lane + 64; b < P.sequences; b += 64) {
      x += value(span_of<kUnit>(P, P.lengths[b]).units);
    }
    return __builtin_amdgcn_readlane(wave_upto(x), 63) * P.heads;
  };
  int const total = over_sequences([](int units) { return units; }), me = (int)blockIdx.x, all = (int)gridDim.x;
  int run = (total + all - 1) / all;
  auto parts_of = [&](int units) { return run == 1 ? units : (units + run - 1) / run; };
  bool apart = over_sequences(parts_of) <= all;
  if (!apart && run >= 8) {  // (an eighth of a run more is less than what a second head costs)
    run++;
    apart = over_sequences(parts_of) <= all;
    run -= apart ? 0 : 1;
  }
  long long const begin = (long long)me * run;
  if (!apart && begin >= total) {
    return;
  }
  int unit = apart ? me : (int)begin;  // (apart: the number of a part)
  int const end = total - unit < run ? total : unit + run;
  int sequence = 0, before = 0, length = 0;  // before: units (parts) of the sequences ahead of it
  for (int base = 0;; base += 64) {
    if (base >= P.sequences) {
      return;  // (fewer parts than workgroups)
    }
    int const b = base + lane, its = base == 0 ? own_length : (b < P.sequences ? P.lengths[b] : 0);
    int units = base == 0 ? own_units : (b < P.sequences ? span_of<kUnit>(P, its).units : 0);
    units = apart ? parts_of(units) : units;
    int const upto = wave_upto(units) * P.heads;
    uint64_t const past = __ballot(before + upto > unit);
    if (past != 0) {
      int const at = __builtin_ctzll(past);
      sequence = base + at;
      length = __builtin_amdgcn_readlane(its, at);
      before += __builtin_amdgcn_readlane(upto - units * P.heads, at);
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  Span span = span_of<kUnit>(P, length);
  int const cuts = apart ? parts_of(span.units) : span.units;
  int head = (unit - before) / cuts, first = (unit - before) - head * cuts, part_index = first;
  int kv = P.row_blocks == 1 ? head : head / P.row_blocks, row_block = head - kv * P.row_blocks;
  int past_it = span.units;  // the unit behind this workgroup's last of the head
  if (apart && cuts > 1) {
    int const each = span.units / cuts, more = span.units - each * cuts;
    first = part_index * each + (part_index < more ? part_index : more);
    past_it = first + each + (part_index < more ? 1 : 0);
  }

  int const R = P.new_tokens * P.group;
  for (;;) {
    int const units = apart ? past_it - first : (span.units - first < end - unit ? span.units - first : end - unit);
    int const row0 = row_block * 16 * RG;
    int const *const table = P.table + (long long)sequence * P.table_width;
    int next_length = 0;  // by a vector load: a scalar one is waited for at once, its register being short
    if (!apart && sequence + 1 < P.sequences) {
      int same = 0;
      asm volatile("" : "+v"(same));
      next_length = P.lengths[sequence + 1 + same];
    }

    // rows: lane's row c of every group, the new token t it belongs to, the keys it sees
    auto query = [&](int row, int d) {  // eight elements of a row of the head, zeros past its end
      uintx4 x = {0, 0, 0, 0};
      if (row < R && d < P.head_dim) {
        int const t = P.new_tokens == 1 ? 0 : quotient(row, P.group, P.group_magic);
        x = *reinterpret_cast<uintx4 const *>(static_cast<T const *>(P.q) + ((long long)sequence * P.new_tokens + t) * P.q_stride +
                                              (long long)(kv * P.group + row - t * P.group) * P.head_dim + d);
      }
      return x;
    };
    auto as_scaled = [&](uintx4 x) { return uintx4{(x[0] & P.q_keep) ^ P.q_flip, (x[1] & P.q_keep) ^ P.q_flip, (x[2] & P.q_keep) ^ P.q_flip, (x[3] & P.q_keep) ^ P.q_flip}; };
    uintx4 q[KK];  // of one group of rows
    int limit[RG], least[RG];
    if constexpr (RG == 1) {
#pragma unroll
      for (int kk = 0; kk < KK; kk++) {
        q[kk] = query(row0 + c, 32 * kk + 8 * g);
      }
    } else {
      for (int i = tid; i < 16 * RG * C; i += kThreads) {
        *reinterpret_cast<uintx4 *>(queries + i / C * (2 * DP) + 16 * place_of<C, false>(i / C, i % C)) = as_scaled(query(row0 + i / C, i % C * 8));
      }
    }
#pragma unroll
    for (int r = 0; r < RG; r++) {
      int const row = row0 + 16 * r + c;
      limit[r] = row < R ? span.to - (P.new_tokens - 1 - (P.new_tokens == 1 ? 0 : quotient(row, P.group, P.group_magic))) : 0;
      least[r] = row < R && P.window != 0 ? limit[r] - P.window : 0;
    }
    // the keys that every row sees lie between these (rows of a block are in the order of their tokens)
    int const last_row = row0 + 16 * RG < R ? row0 + 16 * RG - 1 : R - 1;
    bool const one = P.new_tokens == 1;
    int const all_limit = span.to - (one ? 0 : P.new_tokens - 1 - quotient(row0, P.group, P.group_magic));
    int const all_least = P.window != 0 ? span.to - (one ? 0 : P.new_tokens - 1 - quotient(last_row, P.group, P.group_magic)) - P.window : 0;

    floatx4 acc[RG][DB];
    float m[RG], sum[RG];
#pragma unroll
    for (int r = 0; r < RG; r++) {
      m[r] = -INFINITY;
      sum[r] = 0.0f;
#pragma unroll
      for (int d = 0; d < DB; d++) {
        acc[r][d] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
    // The greatest weight is 2^bias.  2^15 keeps small ones in two words of fp16, and its sums are far from the end of 32 bits.
    // bf16 values reach that end themselves: n weights of at most 2^bias < 1 / 2n add up to less than a half.
    float const bias = std::is_same<T, _Float16>::value ? 15.0f : (float)(__builtin_clz((unsigned)(span.to - span.first) | 1u) - 33);
    uint64_t const k_base = reinterpret_cast<uint64_t>(P.k) + 16ull * kv * P.head_step, v_base = reinterpret_cast<uint64_t>(P.v) + 16ull * kv * P.head_step;

    // as many units at a time as the page numbers in LDS cover
    int const fit = P.page_size < 1 << 16 ? (kIds - 1) * P.page_size / kUnit : 1 << 17;
    for (int part = 0; part < units; part += fit) {
      int const part_units = units - part < fit ? units - part : fit;
      int const key0 = span.from + (first + part) * kUnit, key1 = key0 + part_units * kUnit < span.to ? key0 + part_units * kUnit : span.to;
      int const page0 = quotient(key0, P.page_size, P.page_magic);
      int const numbers = key1 > key0 ? quotient(key1 - 1, P.page_size, P.page_magic) + 1 - page0 : 0;
      __syncthreads();  // (the numbers of the part before, or the tiles as room for sums, are read)
      for (int i = tid; i < numbers; i += kThreads) {
        ids[i] = table[page0 + i];
      }
      if constexpr (RG == 1) {
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {  // the queries are here: no wait for them inside the loop
          q[kk] = part == 0 ? as_scaled(q[kk]) : q[kk];
          asm volatile("" : "+v"(q[kk]));
        }
      }
      __syncthreads();

      // tiles of this wavefront: 32 keys of every unit
      int const mine = key0 + wave * kTile;
      int const tiles = mine < key1 ? (key1 - mine + kUnit - 1) / kUnit : 0;
      uint32_t at[LOADS];     // where the rows begin that this lane loads chunks of, in 16 bytes; all ones: zeros
      uint32_t there = 0;     // keys that exist, a bit each
      auto locate = [&](int tile) {
        int const key = mine + tile * kUnit + lane % kTile;
        int const page = quotient(key, P.page_size, P.page_magic);
        int const number = key >= span.first && key < key1 ? ids[page - page0] : -1;
        bool const is = (unsigned)number < (unsigned)P.pages;
        there = (uint32_t)__ballot(is);
        uint32_t const step = is ? (uint32_t)number * P.page_step + (uint32_t)(key - page * P.page_size) * P.token_step : ~0u;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
          at[i] = (uint32_t)__shfl((int)step, (64 * i + lane) / C, 64);
        }
      };
      auto load = [&](uint64_t base, uint32_t to, auto values) {
        int chunks = P.head_dim / 8;
        asm volatile("" : "+s"(chunks));  // (otherwise a comparison for every load is kept through the loop)
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
          int const row = (64 * i + lane) / C, chunk = chunk_at<C, decltype(values)::value>(row, (64 * i + lane) % C);
          bool const real = at[i] != ~0u && chunk < chunks;
          load_to_lds<PASSING>(real ? base + 16ull * (at[i] + chunk) : reinterpret_cast<uint64_t>(&kZeros), to + 1024 * i);
        }
      };
      using Keys = std::integral_constant<bool, false>;
      using Values = std::integral_constant<bool, true>;

      if (tiles > 0) {
        locate(0);
        load(k_base, k_lds, Keys{});
        load(v_base, v_lds, Values{});
      }
      for (int tile = 0; tile < tiles; tile++) {
        int const key = mine + tile * kUnit;
        uint32_t const is_there = there;
        bool const more = tile + 1 < tiles;
        wait_loads<LOADS>();  // keys are here, values under way

        // S^T: lane has keys 4g .. 4g + 3 and 16 + 4g .. of row c
        floatx4 s[RG][2];
#pragma unroll
        for (int r = 0; r < RG; r++) {
          s[r][0] = s[r][1] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
#pragma unroll
          for (int j = 0; j < 2; j++) {
            int const row = 16 * j + c;
            x8 const k = *reinterpret_cast<x8 const *>(k_tile + row * (2 * DP) + 16 * place_of<C, false>(row, 4 * kk + g));
#pragma unroll
            for (int r = 0; r < RG; r++) {
              if constexpr (RG == 1) {
                s[r][j] = mfma(k, __builtin_bit_cast(x8, q[kk]), s[r][j]);
              } else {
                int const its = 16 * r + c;
                s[r][j] = mfma(k, *reinterpret_cast<x8 const *>(queries + its * (2 * DP) + 16 * place_of<C, false>(its, 4 * kk + g)), s[r][j]);
              }
            }
          }
        }
        wait_lds_reads();
        if (more) {
          locate(tile + 1);
          load(k_base, k_lds, Keys{});
        }

        // weights, as two numbers of the value's type each -- one alone would put as much error into the result as rounding
        // that does
        bool const whole = is_there == ~0u && key >= all_least && key + kTile <= all_limit;
        uintx4 p[RG], rest[RG];
#pragma unroll
        for (int r = 0; r < RG; r++) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            x[e] = s[r][e / 4][e % 4];
          }
          if (!whole) {
            int const upto = limit[r] - key, from = least[r] - key;
            uint32_t seen = is_there;
            seen = upto <= 0 ? 0 : (upto < kTile ? seen & ((1u << upto) - 1) : seen);
            seen = from <= 0 ? seen : (from < kTile ? seen & ~((1u << from) - 1) : 0);
#pragma unroll
            for (int e = 0; e < 8; e++) {
              x[e] = (seen >> (16 * (e / 4) + 4 * g + e % 4)) & 1 ? x[e] : -INFINITY;
            }
          }
          float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
          top = over_groups(top, [](float a, float b) { return fmaxf(a, b); });
          if (__any(top > m[r])) {
            float const higher = fmaxf(m[r], top), less = exp2_fast((m[r] - (higher == -INFINITY ? 0.0f : higher)) * P.scale);
            m[r] = higher;
            sum[r] *= less;
#pragma unroll
            for (int d = 0; d < DB; d++) {
              acc[r][d] *= less;
            }
          }
          float const base = m[r] == -INFINITY ? 0.0f : bias - m[r] * P.scale;
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float const w0 = exp2_fast(__builtin_fmaf(x[e], P.scale, base)), w1 = exp2_fast(__builtin_fmaf(x[e + 1], P.scale, base));
            sum[r] += w0 + w1;
            uint32_t one_pair, its_rest;
            split(w0, w1, one_pair, its_rest, T());
            p[r][e / 2] = one_pair;
            rest[r][e / 2] = its_rest;
          }
        }
        if (more) {
          wait_loads<LOADS>();  // values are here, the next keys under way
        } else {
          wait_loads<0>();
        }

        // Rows of a tile that see other keys than their neighbours: a weight of zero does not keep an infinity or NaN among
        // the values out of a sum.  Such keys' values are added to the rows that do see them by themselves, and zero from
        // then on.
        if (!whole && P.new_tokens > 1) {
          constexpr uint32_t top = Vec<T>::exponent;
          typedef uint16_t shortx2 __attribute__((ext_vector_type(2)));
          shortx2 most = {0, 0};
#pragma unroll
          for (int i = 0; i < LOADS; i++) {
            uintx4 const x = *reinterpret_cast<uintx4 const *>(v_tile + 16 * (64 * i + lane));
#pragma unroll
            for (int w = 0; w < 4; w++) {
              most = __builtin_elementwise_max(most, __builtin_bit_cast(shortx2, x[w] & (top << 16 | top)));
            }
          }
          uint32_t wild = 0;  // keys with such values
          if (__any(most[0] == top || most[1] == top)) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
              uintx4 const x = *reinterpret_cast<uintx4 const *>(v_tile + 16 * (64 * i + lane));
              bool none = false;
#pragma unroll
              for (int w = 0; w < 4; w++) {
                none = none || (x[w] & top) == top || (x[w] & top << 16) == top << 16;
              }
              wild |= none ? 1u << ((64 * i + lane) / C) : 0u;
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
              wild |= (uint32_t)__shfl_xor((int)wild, off, 64);
            }
          }
          for (uint32_t left = __builtin_amdgcn_readfirstlane(wild); left != 0; left &= left - 1) {
            int const j = __builtin_ctz(left), holder = 16 * (j % 16 / 4) + c, at_e = 4 * (j / 16) + j % 4;
            float w[RG];
            bool sees[RG];
#pragma unroll
            for (int r = 0; r < RG; r++) {
              w[r] = 0.0f;
#pragma unroll
              for (int e = 0; e < 8; e++) {
                w[r] = e == at_e ? static_cast<float>(__builtin_bit_cast(x8, p[r])[e]) + static_cast<float>(__builtin_bit_cast(x8, rest[r])[e]) : w[r];
              }
              w[r] = __shfl(w[r], holder, 64);
              sees[r] = key + j < limit[r] && key + j >= least[r];
            }
#pragma unroll
            for (int d = 0; d < DB; d++) {
              x4 const x = *reinterpret_cast<x4 const *>(v_tile + j * (2 * DP) + 16 * place_of<C, true>(j, 2 * d + g / 2) + 8 * (g % 2));
#pragma unroll
              for (int r = 0; r < RG; r++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  acc[r][d][e] += sees[r] ? w[r] * static_cast<float>(x[e]) : 0.0f;
                }
              }
            }
            wait_lds_reads();
            if (lane < C) {
              *reinterpret_cast<uintx4 *>(v_tile + j * (2 * DP) + 16 * lane) = uintx4{0, 0, 0, 0};
            }
          }
        }

        // O^T: lane has columns 16 d + 4g .. + 3 of row c
#pragma unroll
        for (int d = 0; d < DB; d++) {
          uintx2 v[2];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            int const row = 16 * j + 4 * g + c / 4, chunk = 2 * d + c % 4 / 2;
            typedef short shortx4 __attribute__((ext_vector_type(4)));
            unsigned char const *const from = v_tile + row * (2 * DP) + 16 * place_of<C, true>(row, chunk) + 8 * (c % 2);
            v[j] = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (shortx4 __attribute__((address_space(3))) *)(__attribute__((address_space(3))) void const *)from));
          }
          uintx4 const both = {v[0][0], v[0][1], v[1][0], v[1][1]};
          x8 const values = __builtin_bit_cast(x8, both);
#pragma unroll
          for (int r = 0; r < RG; r++) {
            acc[r][d] = mfma(values, __builtin_bit_cast(x8, p[r]), acc[r][d]);
            acc[r][d] = mfma(values, __builtin_bit_cast(x8, rest[r]), acc[r][d]);
          }
        }
        wait_lds_reads();
        if (more) {
          load(v_base, v_lds, Values{});
        }
      }
    }

    // the wavefronts' sums together
    int const rows = R - row0 < 16 * RG ? R - row0 : 16 * RG;
    bool const alone = units == span.units;
    float *const mine = P.parts + (2 * (long long)me + (first == 0 ? 1 : 0)) * part_floats<DP, RG>();
    auto of_sum = [](float all) { return all == 0.0f ? 0.0f : 1.0f / (1.0f + kPart<T>) / all; };
    T *const out = static_cast<T *>(P.out) + (long long)sequence * P.new_tokens * P.out_stride + (long long)kv * P.group * P.head_dim;
    auto store_row = [&](int row, int d, floatx4 x, float by) {  // row of the head, columns d .. d + 3
      if (d < P.head_dim) {
        int const t = P.new_tokens == 1 ? 0 : quotient(row, P.group, P.group_magic);
        x4 y;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          y[e] = static_cast<T>(x[e] * by);
        }
        *reinterpret_cast<x4 *>(out + t * P.out_stride + (row - t * P.group) * P.head_dim + d) = y;
      }
    };
#pragma unroll
    for (int r = 0; r < RG; r++) {
      float const whole_sum = over_groups(sum[r], [](float a, float b) { return a + b; });
      if (g == 0) {
        stat[2 * (wave * 16 * RG + 16 * r + c)] = m[r] * P.scale;
        stat[2 * (wave * 16 * RG + 16 * r + c) + 1] = whole_sum;
      }
    }
    float *const sums = reinterpret_cast<float *>(lds);  // [wave][row][kRow]
    constexpr int kRow = sum_row<DP>();
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RG; r++) {
      int const row = 16 * r + c;
      float its[kWaves][2], top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        its[w][0] = stat[2 * (w * 16 * RG + row)];
        its[w][1] = stat[2 * (w * 16 * RG + row) + 1];
        top = fmaxf(top, its[w][0]);
      }
      float const base = top == -INFINITY ? 0.0f : top, less = exp2_fast(m[r] * P.scale - base);
#pragma unroll
      for (int d = 0; d < DB; d++) {
        *reinterpret_cast<floatx4 *>(sums + (wave * 16 * RG + row) * kRow + 16 * d + 4 * g) = acc[r][d] * less;
      }
      if (wave == r % kWaves && g == 0 && row < rows) {
        float whole_sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
          whole_sum += exp2_fast(its[w][0] - base) * its[w][1];
        }
        row_by[row] = of_sum(whole_sum);
        if (!alone) {
          store_shared(mine + 16 * RG * DP + 4 * row, top, whole_sum);
        }
      }
    }
    __syncthreads();
    for (int i = tid; i < rows * (DP / 4); i += kThreads) {
      int const row = i / (DP / 4), d = i % (DP / 4) * 4;
      floatx4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        x += *reinterpret_cast<floatx4 const *>(sums + (w * 16 * RG + row) * kRow + d);
      }
      if (alone) {
        store_row(row0 + row, d, x, row_by[row]);
      } else {
        store_shared(mine + row * DP + d, x);
      }
    }

    // the last workgroup of a head, or of a group of its parts, joins them
    if (!alone) {
      int const w0 = apart ? me - part_index : (first == 0 ? me : (unit - first) / run), index = me - w0;
      int const count = apart ? cuts : (unit - first + span.units - 1) / run - w0 + 1;
      auto slot = [&](int i) { return P.parts + (2 * (long long)(w0 + i) + (i == 0 ? 1 : 0)) * part_floats<DP, RG>(); };
      auto arrive = [&](int *ticket, int of) {
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        __syncthreads();
        if (tid == 0) {
          int const others = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          *is_last = others == of - 1;
          if (others == of - 1) {
            __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
          }
        }
        __syncthreads();
        return *is_last != 0;
      };
      // Parts i0, i0 + step, .. (n of them), into the first of them or the result; they are asked for together: a trip to the
      // memory that all XCDs share is a microsecond.  A joined part's maximum and sum go beside those it is made of, which
      // other threads may still be reading (level 0 and 2: which of them are read).
      auto join_by = [&](int i0, int step, int n, int level, bool final, auto at_once) {
        constexpr int kBatch = decltype(at_once)::value;
        constexpr int kItems = RG > 1 ? 2 : 1;
        int const items = rows * (DP / 4);
        for (int first_item = tid; first_item < items; first_item += kItems * kThreads) {
          int row[kItems], d[kItems];
          float top[kItems], all_sum[kItems];
          floatx4 x[kItems];
#pragma unroll
          for (int k = 0; k < kItems; k++) {
            int const i = first_item + k * kThreads < items ? first_item + k * kThreads : items - 1;
            row[k] = i / (DP / 4);
            d[k] = i % (DP / 4) * 4;
            top[k] = -INFINITY;
            all_sum[k] = 0.0f;
            x[k] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
          }
          for (int j0 = 0; j0 < n; j0 += kBatch) {
            uint64_t a[kItems][kBatch], b[kItems][kBatch], ms[kItems][kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; j++) {
              float const *const from = slot(i0 + (j0 + j < n ? j0 + j : n - 1) * step);
#pragma unroll
              for (int k = 0; k < kItems; k++) {
                ms[k][j] = load_shared(from + 16 * RG * DP + 4 * row[k] + level);
                a[k][j] = load_shared(from + row[k] * DP + d[k]);
                b[k][j] = load_shared(from + row[k] * DP + d[k] + 2);
              }
            }
#pragma unroll
            for (int j = 0; j < kBatch; j++) {  // (read whether they count or not: under the condition each is a trip of its own)
#pragma unroll
              for (int k = 0; k < kItems; k++) {
                asm volatile("" : "+v"(a[k][j]), "+v"(b[k][j]), "+v"(ms[k][j]));
              }
            }
#pragma unroll
            for (int j = 0; j < kBatch; j++) {
              if (j0 + j < n) {
#pragma unroll
                for (int k = 0; k < kItems; k++) {
                  float const higher = fmaxf(top[k], low_of(ms[k][j])), base = higher == -INFINITY ? 0.0f : higher;
                  float const less = exp2_fast(top[k] - base), its = exp2_fast(low_of(ms[k][j]) - base);
                  top[k] = higher;
                  all_sum[k] = all_sum[k] * less + high_of(ms[k][j]) * its;
                  x[k] = x[k] * less + its * floatx4{low_of(a[k][j]), high_of(a[k][j]), low_of(b[k][j]), high_of(b[k][j])};
                }
              }
            }
          }
#pragma unroll
          for (int k = 0; k < kItems; k++) {
            if (first_item + k * kThreads >= items) {
              break;
            }
            if (final) {
              store_row(row0 + row[k], d[k], x[k], of_sum(all_sum[k]));
            } else {
              store_shared(slot(i0) + row[k] * DP + d[k], x[k]);
              if (d[k] == 0) {
                store_shared(slot(i0) + 16 * RG * DP + 4 * row[k] + 2 - level, top[k], all_sum[k]);
              }
            }
          }
        }
      };
      auto join = [&](int i0, int step, int n, int level, bool final) {  // (what is asked for past the last part is read all the same)
        if (n <= 2) {
          join_by(i0, step, n, level, final, std::integral_constant<int, 2>());
        } else if (n <= 4) {
          join_by(i0, step, n, level, final, std::integral_constant<int, 4>());
        } else {
          join_by(i0, step, n, level, final, std::integral_constant<int, kAtOnce>());
        }
      };
      // in one, two or three levels of groups of up to kAtOnce: a compute unit reads what others wrote at a few bytes a cycle
      int per = count <= kAtOnce ? count : 2;
      while ((count <= kAtOnce * kAtOnce ? per * per : per * per * per) < count) {
        per++;
      }
      for (int at = index, left = count, step = 1, depth = 0;; depth++) {
        int const group = at / per * per, n = left - group < per ? left - group : per;
        bool const final = left <= per;
        // (a workgroup may begin a group of the head that it goes on with, and those of the head that it begins)
        int const ticket = State::kTicketsEach * (w0 + group * step) + (final ? 4 : 2 * depth + (group == 0 ? 0 : 1));
        if (!arrive(P.tickets + State::kJoinStep * ticket, n)) {
          break;
        }
        join(group * step, step, n, depth % 2 * 2, final);
        if (final) {
          break;
        }
        at = group / per;
        left = (left + per - 1) / per;
        step *= per;
      }
    }
    unit += units;
    if (apart || unit >= end) {
      return;
    }
    // the next head begins at its first unit
    first = 0;
    if (++row_block == P.row_blocks) {
      row_block = 0;
      kv++;
    }
    if (unit - before == span.units * P.heads) {
      before = unit;
      sequence++;
      kv = 0;
      span = span_of<kUnit>(P, __builtin_amdgcn_readfirstlane(next_length));
    }
    __syncthreads();  // (`stat`, `is_last` and the tiles are free again)
  }
}

template <class T, int DP, int RG, int WAVES, bool PASSING>
int launch_paged(PagedParams P, int kv_heads) {
  auto *fn = paged_attention_kernel<T, DP, RG, WAVES, PASSING>;
  constexpr int kUnit = kTile * WAVES, lds = lds_bytes<DP, RG, WAVES>(), per_unit = per_compute_unit<DP, RG, WAVES>();
  static_assert(lds <= 160 * 1024, "LDS of a compute unit");
  int const rows = P.new_tokens * P.group;
  P.row_blocks = (rows + 16 * RG - 1) / (16 * RG);
  P.heads = kv_heads * P.row_blocks;
  // workgroups that fit the chip together
  long long const most = (long long)P.sequences * P.heads * (((long long)P.table_width * P.page_size + kUnit - 1) / kUnit + 1);
  long long const room = (long long)(state().scratch_bytes / (2 * part_floats<DP, RG>() * sizeof(float)));
  long long const fit = room < 256LL * per_unit ? room : 256LL * per_unit;
  unsigned const grid = (unsigned)(most < fit ? most : fit);
  if ((size_t)grid * 2 * part_floats<DP, RG>() * sizeof(float) > state().scratch_bytes) {
    return fail(MI355_ERR_INVALID, "mi355_paged_attention: its parts do not fit the workspace");
  }
  MI355_GRANT_LDS(fn, lds);
  MI355_HIP(launch_kernel(fn, dim3(grid), dim3(64 * WAVES), lds, state().stream(), P));
  return MI355_OK;
}

// Two workgroups of four wavefronts to a compute unit, or one of eight: fewer parts to join and, from HBM, wavefronts that
// keep step (of two workgroups the second is served last), but twice the keys to a unit.  Eight where few heads have much
// to read, or all of them more than the caches keep: measured (us, four and eight) 99.7 and 95.7 of 1 sequence x 8 heads x
// 131072 keys, 98.7 and 94.7 of 64 x 8 x 4096, 12.8 and 11.2 of 4 x 8 x 2000, 47.3 and 38.3 of 16 x 4 x 8192 with 32 rows; against it
// 8.8 and 10.4 of 8 x 8 x 500, 32.9 and 38.9 of 128 x 8 x 500, 31.6 and 34.8 of 16 x 8 x 4096, 181 and 222 of 1024 x 8 x 400, and heads
// of 64, of which less is on its way: 37.9 and 41.0 of 47 x 5 x 6280.  With 17 - 48 rows more heads gain, the fewer their keys are
// (us, four and eight, 40 rows of heads of 64): 25.7 and 20.8 of 32 heads x up to 8000 keys, 54.9 and 52.4 of 48 x 30000, 24.8 and 17.9 of
// 96 x 2500, 15.0 and 13.0 of 256 x 500; against it 32.8 and 49.4 of 96 x 8000, 26.2 and 36.9 of 128 x 4000, 21.3 and 31.0 of 256 x 1500,
// 21.6 and 25.4 of 384 x 500.  With 20 rows of heads of 128 the limits lie where these do: 31.2 and 27.7 of 96 x 4000, 17.7 and 15.4 of
// 256 x 500; 37.3 and 40.7 of 128 x 4000, 28.6 and 33.5 of 256 x 1500.
// Eight workgroups of one wavefront for thousands of heads that are short: no wavefront waits for another at a head's end (four
// and one: 93 and 74 us of 1024 sequences x 8 heads x 100 keys, 355 and 244 of 4096 x 8 x 100, 181 and 177 of 1024 x 8 x 400;
// against it 98 and 104 of 64 x 8 x 4096, 33.4 and 33.2 of 128 x 8 x 500, 7.7 and 11.4 of 64 x 8 x 100).
template <class T, int DP, int RG>
int launch_group(PagedParams const &P, int kv_heads, bool passing) {
  if constexpr ((DP <= 128 && RG <= 2) || (DP <= 64 && RG == 3)) {
    long long const heads = (long long)P.sequences * kv_heads * ((P.new_tokens * P.group + 16 * RG - 1) / (16 * RG));
    long long const keys = (long long)P.table_width * P.page_size, units = heads * ((keys + 4 * kTile - 1) / (4 * kTile));
    if constexpr (RG == 1) {
      if (one_wavefront(heads, P.new_tokens * P.group, keys)) {
        return passing ? launch_paged<T, DP, RG, 1, true>(P, kv_heads) : launch_paged<T, DP, RG, 1, false>(P, kv_heads);
      }
    }
    if constexpr (RG <= 2) {
      if (passing && keys >= 1024) {
        return launch_paged<T, DP, RG, (DP <= 64 ? 4 : 8), true>(P, kv_heads);
      }
    }
    bool const few = RG == 1 ? heads <= 96 : heads <= 48 || (heads <= 256 && heads * units <= 300 << 10);
    if (few && units >= 512) {
      return launch_paged<T, DP, RG, 8, false>(P, kv_heads);
    }
  }
  if constexpr (DP > 128) {
    if (passing) {
      return launch_paged<T, DP, RG, 4, true>(P, kv_heads);
    }
  }
  return launch_paged<T, DP, RG, 4, false>(P, kv_heads);
}

template <class T, int DP>
int launch_rows(PagedParams const &P, int kv_heads, bool passing) {
  long long const rows = (long long)P.new_tokens * P.group;
  if (rows <= 16) {
    return launch_group<T, DP, 1>(P, kv_heads, passing);
  }
  if (rows <= 32 || DP > 128) {
    return launch_group<T, DP, 2>(P, kv_heads, passing);
  }
  if constexpr (DP <= 128) {
    return rows <= 48 ? launch_group<T, DP, 3>(P, kv_heads, passing) : launch_group<T, DP, 4>(P, kv_heads, passing);
  }
  return MI355_OK;
}

template <class T>
int launch_head(PagedParams const &P, int kv_heads, bool passing) {
  return P.head_dim <= 64    ? launch_rows<T, 64>(P, kv_heads, passing)
         : P.head_dim <= 96  ? launch_rows<T, 96>(P, kv_heads, passing)
         : P.head_dim <= 128 ? launch_rows<T, 128>(P, kv_heads, passing)
         : P.head_dim <= 192 ? launch_rows<T, 192>(P, kv_heads, passing)
                             : launch_rows<T, 256>(P, kv_heads, passing);
}

}  // namespace paged
}  // namespace mi355
