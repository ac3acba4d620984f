// Log probabilities of given tokens, entropy, and the most probable tokens of rows of logits.
//
// With z_j = scale (x_j - m) and m the greatest logit: log p_j = z_j - log Z, Z = sum e^z_j, and the entropy is
// log Z - (sum z_j e^z_j) / Z, two terms of which neither is below zero.  One pass: a lane keeps the maximum of what it has seen,
// and the two sums relative to it.
//
// The top tokens are found on the way: a wavefront keeps a bound that it knows `top` of its logits to reach, and only logits above
// it are looked at one by one.  The bound is what the top-th of the lanes' own maxima reaches, which the sums need anyway; after the first few
// thousand logits hardly any passes it.  (It is asked for again in nearly every chunk all the same, with more than one top token: the greatest of the lanes' maxima
// of all chunks so far lies above the top-th.)  What passed is told apart by counting: an entry's place is the number of better ones.
//
// Few rows are cut over workgroups, of which the last to come (a ticket) puts the parts together, always in the same order.
//
// Measured: 83 - 86 us of 4096 rows of 50021 fp16 with the top token (410 MB, 4.9 TB/s, and 71 us of vector instructions: a read of so much takes 66),
// 102 with five, 107 with twenty and 124 with fifty, which the bounds take; 143 of fp32 (820 MB, 5.7 TB/s), 11.9 - 13 of 64 rows of 131072 bf16 with
// twenty (17 MB; trips to memory one after the other and the bounds), 22.6 of 200 of these, 7.5 of one row of 32000 fp32 with five, of which a launch is 3.
#include "common.h"
#include "mi355_kernels/kernarg.h"
#include "slices.h"

#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

namespace mi355 {
namespace {

constexpr int kPending = 192;   // tokens that a wavefront has yet to look at; more than 128 are thinned out
constexpr int kGathered = 512;  // entries of a workgroup that are told apart all at once
// Maxima of a lane that bound more than 40 top tokens: what so many of 64 lanes reach rules out little (64 of 131072, 64 rows: 25.6 us with one, 15.3 with
// two, 16.0 with four; 33: 12.3 and 12.8; twenty: 11.7, 12.4 and 14.1).
constexpr int kMaxima = 2;
constexpr int kThreads = 256, kWaves = kThreads / 64, kRounds = 4, kLargestParts = 64;

struct LogParams {
  void const *logits;
  long long stride;
  int const *tokens;
  float *log_probs, *entropy, *top_log_probs;
  int *top_tokens;
  float *parts;  // of each workgroup of a row: maximum, two sums, then the top logits and their tokens
  int *tickets;  // one a row, kJoinStep apart, zero between launches
  int asked, top, vocabulary, row_parts;
  // A difference of logits is that of `part` of each, a half where the scale is below 1: two logits may lie farther apart than 32 bits reach.  The scale of such a
  // difference, times log2 e and as it is.
  float part, scale, natural;
};
constexpr int kPartWords = 4 + 2 * MI355_MAX_TOP;

// x of the lane that the DPP control names
template <int CONTROL>
__device__ __forceinline__ uint32_t moved(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CONTROL, 0xf, 0xf, true); }
// x[l ^ STRIDE]: by moves between registers, where a shuffle is a trip through LDS
template <int STRIDE>
__device__ __forceinline__ uint32_t across(uint32_t x, int lane) {
  if constexpr (STRIDE == 1) {
    return moved<0xb1>(x);  // within fours
  } else if constexpr (STRIDE == 2) {
    return moved<0x4e>(x);
  } else if constexpr (STRIDE == 4) {
    return moved<0x1b>(moved<0x141>(x));  // eights mirrored, then fours
  } else if constexpr (STRIDE == 8) {
    return moved<0x128>(x);  // sixteens turned by eight
  } else {
    uint32_t a = x, b = x;  // (exchanges the odd rows or the upper half of one with the even rows or the lower half of the other)
    if constexpr (STRIDE == 16) {
      asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    } else {
      asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    }
    return (lane & STRIDE) != 0 ? a : b;
  }
}
// over all lanes, in every one; op commutes
template <class Op>
__device__ __forceinline__ float over_lanes(float x, Op op) {
  auto of = [](uint32_t bits) { return __builtin_bit_cast(float, bits); };
  auto bits = [](float v) { return __builtin_bit_cast(uint32_t, v); };
  x = op(x, of(moved<0xb1>(bits(x))));
  x = op(x, of(moved<0x4e>(bits(x))));
  x = op(x, of(moved<0x141>(bits(x))));  // eights, and sixteens, mirrored
  x = op(x, of(moved<0x140>(bits(x))));
  float a = x, b = x;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  a = b = op(a, b);
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return op(a, b);
}

// A logit and its token as one whole number: the better one of two, that with the greater logit or, of equal ones, the lower token, is the greater
// number.  Zero: none.
__device__ __forceinline__ uint32_t ordered(float x) {
  uint32_t const bits = __builtin_bit_cast(uint32_t, x);
  return bits ^ ((int)bits < 0 ? ~0u : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t key) { return __builtin_bit_cast(float, key ^ ((int)key < 0 ? 0x80000000u : ~0u)); }
__device__ __forceinline__ uint64_t entry_of(float x, int token) { return (uint64_t)ordered(x + 0.0f) << 32 | (uint32_t)~token; }  // (no negative zero)
__device__ __forceinline__ float logit_of(uint64_t entry) { return unordered((uint32_t)(entry >> 32)); }
__device__ __forceinline__ int token_of(uint64_t entry) { return (int)~(uint32_t)entry; }

template <int STRIDE>
__device__ __forceinline__ uint64_t across(uint64_t x, int lane) {
  return (uint64_t)across<STRIDE>((uint32_t)(x >> 32), lane) << 32 | across<STRIDE>((uint32_t)x, lane);
}
// Sorts runs of 2 STRIDE lanes that rise and then fall, or the other way round: greatest first, or last.
template <int STRIDE, class T>
__device__ __forceinline__ T cleaned(T x, int lane, bool first) {
  T const other = across<STRIDE>(x, lane);
  x = (other > x) == (((lane & STRIDE) == 0) == first) ? other : x;
  if constexpr (STRIDE > 1) {
    x = cleaned<STRIDE / 2>(x, lane, first);
  }
  return x;
}
template <class T>
__device__ __forceinline__ T sorted(T x, int lane, bool first) {
  x = cleaned<1>(x, lane, (lane & 2) == 0);
  x = cleaned<2>(x, lane, (lane & 4) == 0);
  x = cleaned<4>(x, lane, (lane & 8) == 0);
  x = cleaned<8>(x, lane, (lane & 16) == 0);
  x = cleaned<16>(x, lane, (lane & 32) == 0);
  return cleaned<32>(x, lane, first);
}
// the greatest 64 of a list greatest first and one greatest last, greatest first
__device__ __forceinline__ uint64_t merged(uint64_t a, uint64_t back, int lane) { return cleaned<32>(back > a ? back : a, lane, true); }

// What n of the lanes' values reach, N of a lane (no NaN), and what (n + 3) / 4 do: the upper 16 bits of the n-th greatest, found bit by bit (0.3 us
// of one of a lane; sorting them takes 1.2).
struct Two {
  float nth, earlier;
};
template <int N>
__device__ __forceinline__ Two nth_of_lanes(float const (&value)[N], int n) {
  uint32_t x[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    x[i] = ordered(value[i]);
  }
  auto reach = [&](uint32_t least) {
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      count += __builtin_popcountll(__ballot(x[i] >= least));
    }
    return count;
  };
  uint32_t const lowest = ordered(-INFINITY);
  uint32_t nth = 0, earlier = 0;
#pragma unroll
  for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
    nth = reach(nth | bit) >= n ? nth | bit : nth;
    earlier = reach(earlier | bit) >= (n + 3) / 4 ? earlier | bit : earlier;
  }
  return {unordered(nth > lowest ? nth : lowest), unordered(earlier > lowest ? earlier : lowest)};
}
// the least value above x
__device__ __forceinline__ float above(float x) {
  int const bits = __builtin_bit_cast(int, x + 0.0f);  // (no negative zero)
  return __builtin_bit_cast(float, bits + (bits < 0 ? -1 : 1));
}

// Maximum, sum of 2^z and sum of z 2^z relative to it, z = scale (x - m).
struct Sums {
  float m, s, t;
};
// scale (m - base) for sums that base is to be the maximum of: 0 where there are none yet (nor is there a maximum), and no less than
// -200, whose power is zero as that of minus infinity is, but not a product with it
__device__ __forceinline__ float shift(LogParams const &P, float m, float s, float base) {
  return s == 0.0f ? 0.0f : fmaxf(__builtin_fmaf(m, P.part, -P.part * base) * P.scale, -200.0f);
}
__device__ __forceinline__ Sums moved_to(LogParams const &P, Sums a, float m) {  // m: not below a's
  float const z = shift(P, a.m, a.s, m == -INFINITY ? 0.0f : m), less = __builtin_amdgcn_exp2f(z);
  return {m, a.s * less, less * (a.t + z * a.s)};
}
__device__ __forceinline__ Sums joined(LogParams const &P, Sums a, Sums b) {
  float const m = fmaxf(a.m, b.m);
  a = moved_to(P, a, m);
  b = moved_to(P, b, m);
  return {m, a.s + b.s, a.t + b.t};
}
__device__ __forceinline__ Sums over_lanes(LogParams const &P, Sums a) {
  auto add = [](float x, float y) { return x + y; };
  a = moved_to(P, a, over_lanes(a.m, [](float x, float y) { return fmaxf(x, y); }));
  asm("" : "+v"(a.s), "+v"(a.t));  // (a product fused with the first addition would be rounded in one lane of each two only, and the lanes disagree)
  return {a.m, over_lanes(a.s, add), over_lanes(a.t, add)};
}

__device__ __forceinline__ uint64_t load_shared(float const *p) {
  return __hip_atomic_load((__attribute__((address_space(1))) uint64_t const *)(uint64_t const *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_shared(float *p, uint64_t x) {
  __hip_atomic_store((__attribute__((address_space(1))) uint64_t *)(uint64_t *)p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t both(float x, float y) { return (uint64_t)__builtin_bit_cast(uint32_t, x) | (uint64_t)__builtin_bit_cast(uint32_t, y) << 32; }
__device__ __forceinline__ float low_of(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)x); }

template <class T, bool TOP>
__global__ __launch_bounds__(kThreads) void log_probabilities_kernel(LogParams const P) {
  constexpr int V = 16 / sizeof(T), kChunk = 64 * kRounds * V;
  typedef T piece __attribute__((ext_vector_type(V)));
  __shared__ int pending[kWaves][kPending];  // tokens
  __shared__ uint64_t gathered[kGathered], lists[kWaves][64];
  __shared__ Sums sums[kWaves];
  __shared__ float bounds[kWaves], quarters[kWaves];
  __shared__ int counts[kWaves], count, is_last;
  fetch_kernel_arguments<sizeof(LogParams), 0>();
  int const tid = threadIdx.x, lane = tid % 64, wave = tid / 64, N = P.vocabulary;
  int const part = (int)(blockIdx.x % (unsigned)P.row_parts);
  long long const row = blockIdx.x / (unsigned)P.row_parts;
  T const *const logits = static_cast<T const *>(P.logits) + row * P.stride;

  // Pieces of 16 bytes at multiples of 16: `ahead` elements before the row's first are not its own.
  int const ahead = (int)((reinterpret_cast<uintptr_t>(logits) % 16) / sizeof(T));
  int const chunks = (int)(((long long)N + ahead + kChunk - 1) / kChunk), all_waves = P.row_parts * kWaves;
  struct Held {
    piece x[kRounds];
  };
  auto first_of = [&](int chunk) { return chunk * kChunk - ahead; };  // (the vocabulary is at most 2^30)
  auto hold = [&](int chunk) {
    Held h;
    int const j0 = first_of(chunk);
    if (j0 >= 0 && j0 + kChunk <= N) {
#pragma unroll
      for (int r = 0; r < kRounds; r++) {
        h.x[r] = *reinterpret_cast<piece const *>(logits + j0 + (64 * r + lane) * V);
      }
    } else {
      // A row's first and last chunk: pieces that lie in the row whole are asked for as ever (in the place of others the first such one), of
      // those that do in part, one at either end, each element.
      bool const some = N >= 2 * V;
#pragma unroll
      for (int r = 0; r < kRounds; r++) {
        int const j = j0 + (64 * r + lane) * V, first = ahead == 0 ? 0 : V - ahead;
        h.x[r] = some ? *reinterpret_cast<piece const *>(logits + (j >= 0 && j <= N - V ? j : first)) : piece{};
      }
#pragma unroll
      for (int r = 0; r < kRounds; r++) {
        int const j = j0 + (64 * r + lane) * V;
        if (!some || j < 0 || j > N - V) {
#pragma unroll
          for (int e = 0; e < V; e++) {
            h.x[r][e] = static_cast<T>(-INFINITY);
          }
          if (j > -V && j < N) {
#pragma unroll
            for (int e = 0; e < V; e++) {
              h.x[r][e] = j + e >= 0 && j + e < N ? logits[j + e] : static_cast<T>(-INFINITY);
            }
          }
        }
      }
    }
    return h;
  };
  // the tokens asked for, on their way while the row is read (whoever comes last has them)
  float asked_x = -INFINITY;
  if (wave == 0 && lane < P.asked) {
    int const token = P.tokens[row * P.asked + lane];
    asked_x = token >= 0 && token < N ? static_cast<float>(logits[token]) : -INFINITY;
  }

  Sums own = {-INFINITY, 0.0f, 0.0f};
  float maxima[kMaxima] = {-INFINITY, -INFINITY};  // of the halves of what a lane sees of each chunk
  float bound = -INFINITY, quarter = -INFINITY;  // that as many as asked for, and a quarter of these, reach
  int waiting = 0;    // tokens of this wavefront's that may be among the top ones
  uint64_t best = 0;  // the best of those that were thinned out, a lane each, best first
  auto waiting_entry = [&](int i) {  // (their logits are read again: finding them again in registers takes longer)
    int const token = i < waiting ? pending[wave][i] : 0;
    return i < waiting ? entry_of(static_cast<float>(logits[token]), token) : 0;
  };
  auto thin = [&]() {  // the first 64
    best = merged(best, sorted(waiting_entry(lane), lane, false), lane);
    int const second = pending[wave][64 + lane], third = pending[wave][128 + lane];
    pending[wave][lane] = second;
    pending[wave][64 + lane] = third;
    waiting = waiting > 64 ? waiting - 64 : 0;
  };
  int chunk = part * kWaves + wave;
  if (chunk < chunks) {
    Held next = hold(chunk);
    for (; chunk < chunks; chunk += all_waves) {
      Held const h = next;
      if (chunk + all_waves < chunks) {
        next = hold(chunk + all_waves);
      }
      float x[kRounds * V], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < kMaxima; j++) {
#pragma unroll
        for (int i = j * (kRounds * V / kMaxima); i < (j + 1) * (kRounds * V / kMaxima); i++) {
          x[i] = static_cast<float>(h.x[i / V][i % V]);
          maxima[j] = fmaxf(maxima[j], x[i]);
        }
        top = fmaxf(top, maxima[j]);
      }
      own = moved_to(P, own, top);
      float const base = own.m == -INFINITY ? 0.0f : -P.part * own.m;
      float s = 0.0f, t = 0.0f;
#pragma unroll
      for (int i = 0; i < kRounds * V; i++) {
        // (the difference first: the product of a large maximum would be off by more than the lanes' maxima differ)
        float const z = __builtin_fmaf(x[i], P.part, base) * P.scale, w = __builtin_amdgcn_exp2f(z);
        s += w;
        t = __builtin_fmaf(fmaxf(z, -200.0f), w, t);  // (2^-200 is zero: a z of minus infinity would make it NaN)
      }
      own.s += s;
      own.t += t;
      if constexpr (TOP) {
        if (__any(top > bound)) {
          // (an element that equals an earlier bound comes behind as many that are no less)
          Two reached;
          if (P.top == 1) {
            reached.nth = reached.earlier = over_lanes(top, [](float x, float y) { return fmaxf(x, y); });
          } else if (P.top <= 40) {
            float const most[1] = {top};
            reached = nth_of_lanes(most, P.top);
          } else {
            reached = nth_of_lanes(maxima, P.top);
          }
          float const least = reached.nth > bound ? reached.nth : above(bound);
          bound = fmaxf(bound, reached.nth);
          quarter = reached.earlier;
          int const j0 = first_of(chunk) + lane * V;
          uint32_t passing = 0;
#pragma unroll
          for (int i = 0; i < kRounds * V; i++) {
            passing |= x[i] >= least ? 1u << i : 0u;
          }
          for (uint64_t which = __ballot(passing != 0); which != 0; which = __ballot(passing != 0)) {
            if (passing != 0) {
              int const i = __builtin_ctz(passing);
              int const place = waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(which >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)which, 0));
              pending[wave][place] = j0 + 64 * V * (i / V) + i % V;
              passing &= passing - 1;
            }
            waiting += __builtin_popcountll(which);
            if (waiting > 128) {
              thin();
            }
          }
        }
      }
    }
  }

  // The wavefronts' sums together, and their entries that no bound rules out.
  own = over_lanes(P, own);
  if (lane == 0) {
    sums[wave] = own;
    bounds[wave] = bound;
    quarters[wave] = quarter;
  }
  if (tid == 0) {
    count = 0;
  }
  // Puts those of N entries a lane that reach the bound into `gathered`; more than fit are counted only.
  auto gather = [&](auto n, auto const &its) {
    constexpr int kN = decltype(n)::value;
    int total = 0, before[kN];
    uint64_t which[kN];
    uint64_t const least = (uint64_t)ordered(bound > -INFINITY ? bound + 0.0f : above(bound)) << 32;
#pragma unroll
    for (int i = 0; i < kN; i++) {
      which[i] = __ballot(its[i] >= least);
      before[i] = total;
      total += __builtin_popcountll(which[i]);
    }
    if (total != 0) {
      int base = 0;
      if (lane == 0) {
        base = __hip_atomic_fetch_add(&count, total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
      for (int i = 0; i < kN; i++) {
        int const place = base + before[i] + __builtin_amdgcn_mbcnt_hi((uint32_t)(which[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)which[i], 0));
        if ((which[i] >> lane & 1) != 0 && place < kGathered) {
          gathered[place] = its[i];
        }
      }
    }
  };
  // put(place, entry) for the `top` best of those gathered, by the thread that has it, best first, and none behind them.  How many are better
  // is an entry's place: a few instructions for each two of them, where sorting takes 140 cycles for each of 21 steps.
  auto place_gathered = [&](auto put) {
    int const n = count;
    for (int mine = tid; mine < n; mine += kThreads) {
      uint64_t const entry = gathered[mine];
      int place = 0;
      int j = 0;
      for (; j + 8 <= n; j += 8) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          place += gathered[j + i] > entry ? 1 : 0;
        }
      }
      for (; j < n; j++) {
        place += gathered[j] > entry ? 1 : 0;
      }
      if (place < P.top) {
        put(place, entry);
      }
    }
    if (tid >= n && tid < P.top) {
      put(tid, 0);
    }
  };
  auto place_lists = [&](auto put) {  // the same of the wavefronts' `best`
    lists[wave][63 - lane] = best;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; w++) {
        best = merged(best, lists[w][lane], lane);
      }
      if (lane < P.top) {
        put(lane, best);
      }
    }
  };
  __syncthreads();
  own = joined(P, joined(P, sums[0], sums[1]), joined(P, sums[2], sums[3]));
  if constexpr (TOP) {
    static_assert(kWaves == 4, "sums and bounds");
    bound = fmaxf(fmaxf(bounds[0], bounds[1]), fmaxf(bounds[2], bounds[3]));
    bound = fmaxf(bound, fminf(fminf(quarters[0], quarters[1]), fminf(quarters[2], quarters[3])));
    uint64_t const its[3] = {lane < P.top ? best : 0, waiting_entry(lane), waiting_entry(64 + lane)};
    gather(std::integral_constant<int, 3>(), its);
    __syncthreads();
  }
  auto place_own = [&](auto put) {
    if (count <= kGathered) {
      place_gathered(put);
    } else {
      while (waiting > 0) {
        thin();
      }
      place_lists(put);
    }
  };

  auto answer = [&](auto place) {
    constexpr float kLn2 = 0.693147180559945309f;
    bool const empty = own.m == -INFINITY && own.s == 0.0f, wild = !(own.s < INFINITY) || own.m == INFINITY;
    float const log_z = log2f(own.s), nan = __builtin_nanf("");
    auto log_of = [&](float x) {
      // (in natural units from the start: a token masked by the type's lowest value has a log probability that 32 bits hold, and log2 e times it passes them)
      return wild ? nan : (empty || x == -INFINITY ? -INFINITY : __builtin_fmaf(x, P.part, -P.part * own.m) * P.natural - kLn2 * log_z);
    };
    if (wave == 0) {
      for (int i = lane; i < P.asked; i += 64) {
        if (i >= 64) {
          int const token = P.tokens[row * P.asked + i];
          asked_x = token >= 0 && token < N ? static_cast<float>(logits[token]) : -INFINITY;
        }
        P.log_probs[row * P.asked + i] = log_of(asked_x);
      }
      if (lane == 0) {
        P.entropy[row] = wild ? nan : (empty ? 0.0f : kLn2 * (log_z - own.t / own.s));
      }
    }
    if constexpr (TOP) {
      place([&](int i, uint64_t entry) {
        bool const is = entry != 0 && !wild;
        P.top_log_probs[row * P.top + i] = wild ? nan : (is ? log_of(logit_of(entry)) : -INFINITY);
        P.top_tokens[row * P.top + i] = is ? token_of(entry) : -1;
      });
    }
  };
  if (P.row_parts == 1) {
    answer(place_own);
    return;
  }

  float *const mine = P.parts + (long long)blockIdx.x * kPartWords;
  if (tid == 0) {
    store_shared(mine, both(own.m, own.s));
    store_shared(mine + 2, both(own.t, 0.0f));
  }
  if constexpr (TOP) {
    place_own([&](int i, uint64_t entry) { store_shared(mine + 4 + 2 * i, entry); });
  }
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  __syncthreads();
  if (tid == 0) {
    int *const ticket = P.tickets + row * State::kJoinStep;
    is_last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == P.row_parts - 1;
    if (is_last) {
      __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
    }
    count = 0;
  }
  __syncthreads();
  if (!is_last) {
    return;
  }
  // Every wavefront has the sums of all parts, and the lists of some, four at a time; what their last ones reach rules out most of the others.
  float const *const parts = P.parts + row * P.row_parts * kPartWords;
  static_assert(kLargestParts <= 64, "a lane has a part");
  constexpr int kEach = 4;
  auto ask = [&](int first, uint64_t (&its)[kEach]) {  // best last
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      int const which = first + wave + i * kWaves;
      its[i] = load_shared(parts + (which < P.row_parts ? which : 0) * kPartWords + 4 + 2 * (63 - lane < P.top ? 63 - lane : 0));
    }
  };
  auto only_theirs = [&](int first, uint64_t (&its)[kEach]) {
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      its[i] = first + wave + i * kWaves < P.row_parts && 63 - lane < P.top ? its[i] : 0;
    }
  };
  uint64_t its[kEach], ends = 0, earlier = 0;
  float const *const its_part = parts + (lane < P.row_parts ? lane : 0) * kPartWords;
  uint64_t const m_s = load_shared(its_part), t = load_shared(its_part + 2);
  if constexpr (TOP) {
    ends = load_shared(its_part + 4 + 2 * (P.top - 1));
    earlier = load_shared(its_part + 4 + 2 * ((P.top - 1) / P.row_parts));
    ask(0, its);
  }
  own = lane < P.row_parts ? Sums{low_of(m_s), low_of(m_s >> 32), low_of(t)} : Sums{-INFINITY, 0.0f, 0.0f};
  own = over_lanes(P, own);
  if constexpr (TOP) {
    // what every list's last one reaches, and what its share of them does
    auto reached = [](uint64_t entry) { return entry != 0 ? logit_of(entry) : -INFINITY; };
    bound = over_lanes(lane < P.row_parts ? reached(ends) : -INFINITY, [](float x, float y) { return fmaxf(x, y); });
    bound = fmaxf(bound, over_lanes(lane < P.row_parts ? reached(earlier) : INFINITY, [](float x, float y) { return fminf(x, y); }));
    for (int first = 0; first < P.row_parts; first += kEach * kWaves) {
      if (first > 0) {
        ask(first, its);
      }
      only_theirs(first, its);
      gather(std::integral_constant<int, kEach>(), its);
    }
    __syncthreads();
  }
  answer([&](auto put) {
    if (count <= kGathered) {
      place_gathered(put);
    } else {
      best = 0;
      for (int first = 0; first < P.row_parts; first += kEach * kWaves) {
        ask(first, its);
        only_theirs(first, its);
#pragma unroll
        for (int i = 0; i < kEach; i++) {
          best = merged(best, its[i], lane);
        }
      }
      place_lists(put);
    }
  });
}

template <class T>
int launch_log(LogParams P, int rows) {
  constexpr int kChunk = 64 * kRounds * (16 / (int)sizeof(T));
  // As many workgroups to a row as leave two to a compute unit, each with a chunk for every wavefront at least.  Measured (us, one, two and four to a
  // compute unit; 131072 bf16 a row, 20 top tokens): 13.4, 11.9 and 12.9 of 64 rows, 24.1, 22.7 and 23.9 of 200; alike for few rows.
  constexpr int kFill = 512;
  int const most = (P.vocabulary - 1) / (kWaves * kChunk) + 1, wanted = rows < kFill ? (kFill - 1) / rows + 1 : 1;
  P.row_parts = wanted < most ? wanted : most;
  P.row_parts = P.row_parts < kLargestParts ? P.row_parts : kLargestParts;
  auto *fn = P.top > 0 ? log_probabilities_kernel<T, true> : log_probabilities_kernel<T, false>;
  return in_slices(rows, 1 << 22, [&](long long at, long long count) -> int {
    LogParams Q = P;
    Q.logits = static_cast<T const *>(P.logits) + at * P.stride;
    Q.tokens = P.tokens != nullptr ? P.tokens + at * P.asked : nullptr;
    Q.log_probs = P.log_probs != nullptr ? P.log_probs + at * P.asked : nullptr;
    Q.entropy = P.entropy + at;
    Q.top_log_probs = P.top > 0 ? P.top_log_probs + at * P.top : nullptr;
    Q.top_tokens = P.top > 0 ? P.top_tokens + at * P.top : nullptr;
    MI355_HIP(launch_kernel(fn, dim3((unsigned)(count * P.row_parts)), dim3(kThreads), 0, state().stream(), Q));
    return MI355_OK;
  });
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355_log_probabilities(void const *logits, long long stride, int const *tokens, float *log_probs, float *entropy,
                                       float *top_log_probs, int *top_tokens, int rows, int asked, int top, int vocabulary, float scale,
                                       int type) {
  MI355_REQUIRE_INIT();
  if (rows < 0 || asked < 0 || top < 0 || vocabulary < 1 || !(scale > 0.0f) || !std::isfinite(scale) || (rows > 1 && stride < vocabulary)) {
    return fail(MI355_ERR_INVALID, "mi355_log_probabilities: %d rows of %d, %lld apart, %d asked for, %d top ones, scale %g", rows, vocabulary,
                stride, asked, top, (double)scale);
  }
  if (type != MI355_TYPE_F16 && type != MI355_TYPE_BF16 && type != MI355_TYPE_F32) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_log_probabilities: type %d", type);
  }
  if (top > MI355_MAX_TOP || vocabulary > MI355_MAX_VOCABULARY) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_log_probabilities: %d top tokens of %d", top, vocabulary);
  }
  if (rows == 0) {
    return MI355_OK;
  }
  if (logits == nullptr || entropy == nullptr || (asked > 0 && (tokens == nullptr || log_probs == nullptr)) ||
      (top > 0 && (top_log_probs == nullptr || top_tokens == nullptr))) {
    return fail(MI355_ERR_INVALID, "mi355_log_probabilities: null pointer");
  }
  if (reinterpret_cast<uintptr_t>(logits) % (type == MI355_TYPE_F32 ? 4 : 2) != 0) {
    return fail(MI355_ERR_INVALID, "mi355_log_probabilities: logits begin between two elements");
  }
  State &s = state();
  float const part = scale < 1.0f ? 0.5f : 1.0f, natural = scale / part;
  LogParams const P{logits, stride, tokens, log_probs, entropy, top_log_probs, top_tokens, static_cast<float *>(s.scratch()), s.queue_join_tickets(),
                    asked, top, vocabulary, 1, part, fminf(natural * 1.44269504088896341f, FLT_MAX), natural};
  return type == MI355_TYPE_F16 ? launch_log<_Float16>(P, rows) : type == MI355_TYPE_BF16 ? launch_log<__bf16>(P, rows) : launch_log<float>(P, rows);
}
