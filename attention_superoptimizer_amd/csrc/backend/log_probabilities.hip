// Log probabilities of given tokens, entropy, and the most probable tokens of rows of logits.
//
// With z_j = scale (x_j - m) and m the greatest logit: log p_j = z_j - log Z, Z = sum e^z_j, and the entropy is
// log Z - (sum z_j e^z_j) / Z, two terms of which neither is below zero.  One pass: a lane keeps the maximum of what it has seen,
// and the two sums relative to it.
//
// The top tokens are found on the way: a wavefront keeps a bound that it knows `top` of its logits to reach, and only logits above
// it are looked at one by one.  The bound is the top-th of the lanes' own maxima, which the sums need anyway; after the first few
// thousand logits hardly any passes it.
#include "common.h"
#include "mi355_kernels/kernarg.h"
#include "slices.h"

#include <climits>
#include <cmath>

namespace mi355 {
namespace {

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
  float scale;  // times log2 e
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

// A logit and its token; the better one of two is the greater, of equal ones the one with the lower token.
struct Entry {
  float x;
  int token;
};
__device__ __forceinline__ Entry none() { return {-INFINITY, INT_MAX}; }
__device__ __forceinline__ bool better(Entry a, Entry b) { return a.x > b.x || (a.x == b.x && a.token < b.token); }
// towards best first, or last
template <int STRIDE>
__device__ __forceinline__ Entry exchanged(Entry e, int lane, bool first) {
  Entry const other = {__builtin_bit_cast(float, across<STRIDE>(__builtin_bit_cast(uint32_t, e.x), lane)), (int)across<STRIDE>((uint32_t)e.token, lane)};
  return better(other, e) == (((lane & STRIDE) == 0) == first) ? other : e;
}
template <int STRIDE>
__device__ __forceinline__ Entry cleaned(Entry e, int lane, bool first) {
  e = exchanged<STRIDE>(e, lane, first);
  if constexpr (STRIDE > 1) {
    e = cleaned<STRIDE / 2>(e, lane, first);
  }
  return e;
}
// from any order to best last
__device__ __forceinline__ Entry sorted_back(Entry e, int lane) {
  e = cleaned<1>(e, lane, (lane & 2) == 0);
  e = cleaned<2>(e, lane, (lane & 4) == 0);
  e = cleaned<4>(e, lane, (lane & 8) == 0);
  e = cleaned<8>(e, lane, (lane & 16) == 0);
  e = cleaned<16>(e, lane, (lane & 32) == 0);
  return cleaned<32>(e, lane, false);
}
// the best 64 of a list best first and one best last, best first
__device__ __forceinline__ Entry merged(Entry a, Entry back, int lane) { return cleaned<32>(better(back, a) ? back : a, lane, true); }

// The n-th greatest of the lanes' values (n <= 64; no NaN), bit by bit of an order-preserving whole number, of which a T has the upper BITS.
template <int BITS>
__device__ __forceinline__ float nth_of_lanes(float x, int n) {
  uint32_t const bits = __builtin_bit_cast(uint32_t, x), key = bits ^ ((int)bits < 0 ? ~0u : 0x80000000u);
  uint32_t found = 0;
#pragma unroll
  for (int bit = 31; bit >= 32 - BITS; bit--) {
    uint32_t const with = found | 1u << bit;
    found = __builtin_popcountll(__ballot(key >= with)) >= n ? with : found;
  }
  found |= (int)found < 0 ? 0 : (BITS < 32 ? (1u << (32 - BITS)) - 1 : 0);  // (of a negative value the lower bits are ones)
  return __builtin_bit_cast(float, found ^ ((int)found < 0 ? 0x80000000u : ~0u));
}

// Maximum, sum of 2^z and sum of z 2^z relative to it, z = scale (x - m).
struct Sums {
  float m, s, t;
};
// scale (m - base) for sums that base is to be the maximum of: 0 where there are none yet (nor is there a maximum), and no less than
// -200, whose power is zero as that of minus infinity is, but not a product with it
__device__ __forceinline__ float shift(float m, float s, float base, float scale) { return s == 0.0f ? 0.0f : fmaxf((m - base) * scale, -200.0f); }
__device__ __forceinline__ Sums moved_to(Sums a, float m, float scale) {  // m: not below a's
  float const z = shift(a.m, a.s, m == -INFINITY ? 0.0f : m, scale), less = __builtin_amdgcn_exp2f(z);
  return {m, a.s * less, less * (a.t + z * a.s)};
}
__device__ __forceinline__ Sums joined(Sums a, Sums b, float scale) {
  float const m = fmaxf(a.m, b.m);
  a = moved_to(a, m, scale);
  b = moved_to(b, m, scale);
  return {m, a.s + b.s, a.t + b.t};
}
__device__ __forceinline__ Sums over_lanes(Sums a, float scale) {
  auto add = [](float x, float y) { return x + y; };
  a = moved_to(a, over_lanes(a.m, [](float x, float y) { return fmaxf(x, y); }), scale);
  return {a.m, over_lanes(a.s, add), over_lanes(a.t, add)};
}

__device__ __forceinline__ uint64_t load_shared(float const *p) {
  return __hip_atomic_load((__attribute__((address_space(1))) uint64_t const *)(uint64_t const *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_shared(float *p, float x, uint32_t y) {
  __hip_atomic_store((__attribute__((address_space(1))) uint64_t *)(uint64_t *)p, (uint64_t)__builtin_bit_cast(uint32_t, x) | (uint64_t)y << 32, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float low_of(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)x); }

template <class T, bool TOP>
__global__ __launch_bounds__(kThreads) void log_probabilities_kernel(LogParams const P) {
  constexpr int V = 16 / sizeof(T), kChunk = 64 * kRounds * V;
  typedef T piece __attribute__((ext_vector_type(V)));
  __shared__ Entry pending[kWaves][128];
  __shared__ Entry lists[kWaves][64];
  __shared__ Sums sums[kWaves];
  __shared__ int is_last;
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
  Entry best = none();
  float bound = -INFINITY;
  int waiting = 0;  // entries of this wavefront's that are not in `best` yet
  auto take = [&](int n) {
    best = merged(best, sorted_back(lane < n ? pending[wave][lane] : none(), lane), lane);
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
      for (int i = 0; i < kRounds * V; i++) {
        x[i] = static_cast<float>(h.x[i / V][i % V]);
        top = fmaxf(top, x[i]);
      }
      own = moved_to(own, fmaxf(own.m, top), P.scale);
      float const base = own.m == -INFINITY ? 0.0f : own.m;
      float s = 0.0f, t = 0.0f;
#pragma unroll
      for (int i = 0; i < kRounds * V; i++) {
        // (the difference first: the product of a large maximum would be off by more than the lanes' maxima differ)
        float const z = (x[i] - base) * P.scale, w = __builtin_amdgcn_exp2f(z);
        s += w;
        t = __builtin_fmaf(fmaxf(z, -200.0f), w, t);  // (2^-200 is zero: a z of minus infinity would make it NaN)
      }
      own.s += s;
      own.t += t;
      if constexpr (TOP) {
        if (__any(top > bound)) {
          float const before = bound, reached = nth_of_lanes<(sizeof(T) == 4 ? 32 : __is_same(T, _Float16) ? 19 : 16)>(own.m, P.top);
          bound = fmaxf(bound, reached);
          int const j0 = first_of(chunk) + lane * V;
#pragma unroll
          for (int i = 0; i < kRounds * V; i++) {
            bool const passes = x[i] > before && x[i] >= bound;
            uint64_t const which = __ballot(passes);
            if (which != 0) {
              if (passes) {
                int const place = waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(which >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)which, 0));
                pending[wave][place] = {x[i], j0 + 64 * V * (i / V) + i % V};
              }
              waiting += __builtin_popcountll(which);
              if (waiting > 64) {
                take(64);
                waiting -= 64;
                Entry const e = pending[wave][64 + lane];
                pending[wave][lane] = e;
              }
            }
          }
        }
      }
    }
  }

  // the wavefront's, then the workgroup's
  own = over_lanes(own, P.scale);
  if constexpr (TOP) {
    if (waiting > 0) {
      take(waiting);
    }
    lists[wave][63 - lane] = best;
  }
  if (lane == 0) {
    sums[wave] = own;
  }
  auto join_waves = [&]() {  // by the first wavefront
    own = sums[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) {
      own = joined(own, sums[w], P.scale);
      if constexpr (TOP) {
        best = merged(best, lists[w][lane], lane);
      }
    }
  };
  __syncthreads();
  if (wave == 0) {
    join_waves();
  }
  if (P.row_parts > 1) {
    float *const mine = P.parts + (long long)blockIdx.x * kPartWords;
    if (wave == 0) {
      if (lane == 0) {
        store_shared(mine, own.m, __builtin_bit_cast(uint32_t, own.s));
        store_shared(mine + 2, own.t, 0);
      }
      if (TOP && lane < P.top) {
        store_shared(mine + 4 + 2 * lane, best.x, (uint32_t)best.token);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    __syncthreads();
    if (tid == 0) {
      int *const ticket = P.tickets + row * State::kJoinStep;
      is_last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == P.row_parts - 1;
      if (is_last) {
        __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
      }
    }
    __syncthreads();
    if (!is_last) {
      return;
    }
    float const *const parts = P.parts + row * P.row_parts * kPartWords;
    own = {-INFINITY, 0.0f, 0.0f};
    if (tid < P.row_parts) {
      uint64_t const m_s = load_shared(parts + tid * kPartWords), t = load_shared(parts + tid * kPartWords + 2);
      own = {low_of(m_s), __builtin_bit_cast(float, (uint32_t)(m_s >> 32)), low_of(t)};
    }
    if constexpr (TOP) {
      constexpr int kEach = kLargestParts / kWaves;
      uint64_t its[kEach];  // all lists of this wavefront's parts, best last, asked for together
#pragma unroll
      for (int i = 0; i < kEach; i++) {
        int const part_i = wave + i * kWaves;
        if (i * kWaves < P.row_parts) {
          its[i] = load_shared(parts + (part_i < P.row_parts ? part_i : 0) * kPartWords + 4 + 2 * (63 - lane < P.top ? 63 - lane : 0));
        }
      }
      best = none();
#pragma unroll
      for (int i = 0; i < kEach; i++) {
        if (wave + i * kWaves < P.row_parts) {
          best = merged(best, 63 - lane < P.top ? Entry{low_of(its[i]), (int)(its[i] >> 32)} : none(), lane);
        }
      }
      lists[wave][63 - lane] = best;
    }
    own = over_lanes(own, P.scale);
    if (lane == 0) {
      sums[wave] = own;
    }
    __syncthreads();
    if (wave == 0) {
      join_waves();
    }
  }
  if (wave != 0) {
    return;
  }

  constexpr float kLn2 = 0.693147180559945309f;
  bool const empty = own.m == -INFINITY && own.s == 0.0f, wild = !(own.s < INFINITY) || own.m == INFINITY;
  float const log_z = log2f(own.s), nan = __builtin_nanf("");
  auto log_of = [&](float x) {
    return wild ? nan : (empty || x == -INFINITY ? -INFINITY : kLn2 * ((x - own.m) * P.scale - log_z));
  };
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
  if (TOP && lane < P.top) {
    bool const is = best.x > -INFINITY && !wild;
    P.top_log_probs[row * P.top + lane] = is || wild ? log_of(best.x) : -INFINITY;
    P.top_tokens[row * P.top + lane] = is ? best.token : -1;
  }
}

template <class T>
int launch_log(LogParams P, int rows) {
  constexpr int kChunk = 64 * kRounds * (16 / (int)sizeof(T));
  // As many workgroups to a row as fill the chip four times over, each with a chunk for every wavefront at least.
  int const most = (P.vocabulary - 1) / (kWaves * kChunk) + 1, wanted = rows < 1024 ? (1023 / rows) + 1 : 1;
  P.row_parts = wanted < most ? wanted : most;
  P.row_parts = P.row_parts < kLargestParts ? P.row_parts : kLargestParts;
  auto *fn = P.top > 0 ? log_probabilities_kernel<T, true> : log_probabilities_kernel<T, false>;
  return in_slices(rows, (1 << 30) / kLargestParts, [&](long long at, long long count) -> int {
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
  LogParams const P{logits, stride, tokens, log_probs, entropy, top_log_probs, top_tokens, static_cast<float *>(s.scratch()), s.queue_join_tickets(),
                    asked, top, vocabulary, 1, scale * 1.44269504088896341f};
  return type == MI355_TYPE_F16 ? launch_log<_Float16>(P, rows) : type == MI355_TYPE_BF16 ? launch_log<__bf16>(P, rows) : launch_log<float>(P, rows);
}
