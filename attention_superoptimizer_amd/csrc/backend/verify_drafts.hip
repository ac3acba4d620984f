// Speculative sampling's decision about drafted tokens.
//
// Draft i stays while u_i q_i(x_i) < p_i(x_i): the product of two 24-bit numbers is exact in 64 bits.  The next token is
// the lowest j whose sum of weights w_0 + .. + w_j passes u times their total, summed in 64 bits: among 10^5 weights
// 32-bit sums would be off by whole tokens.
//
// What has to be read is one row of p and one of q a sequence, at a place that is known after two trips to memory (the
// drafted tokens, their probabilities).  A row is cut into strips of a few hundred or thousand tokens, a wavefront's each, so
// that one sequence, too, is read by many compute units; every wavefront finds the place by itself, adds up its strips and
// leaves their sums, and the last workgroup of a sequence (a ticket) finds the strip that holds the token and reads that one
// again.  Sums are added in an order that does not depend on who comes last.  Bound by HBM for a batch (64 sequences x 131072
// fp32, 67 MB: 16 us, 4.2 TB/s), by the chain of trips for one sequence (5.4 us).
#include "common.h"
#include "slices.h"

#include <climits>
#include <cmath>

namespace mi355 {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

struct VerifyParams {
  void const *target, *draft;
  int const *tokens;
  float const *uniforms;
  int *accepted, *out;
  double *parts;  // two sums of every strip
  int *tickets;   // one a sequence, kJoinStep apart, zero between launches
  int drafts, vocabulary, strips, each;  // strips of a row, and how many a wavefront has
};

// x of the lane that the DPP control names, zero where there is none (rows that ROWS leaves out get zero too)
template <int CONTROL, int ROWS>
__device__ __forceinline__ double moved(double x) {
  uint64_t const bits = __builtin_bit_cast(uint64_t, x);
  uint32_t const low = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, CONTROL, ROWS, 0xf, true);
  uint32_t const high = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), CONTROL, ROWS, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)low | (uint64_t)high << 32);
}
// The sum of the lanes up to this one: within rows of 16, then the ends of rows.  Moves between registers: the same by
// shuffles, each a trip through LDS, had this kernel wait for 10 us of its 17 for one sequence.
__device__ __forceinline__ double wave_upto(double x) {
  x += moved<0x111, 0xf>(x);  // from 1, 2, 4, 8 lanes before in the row
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);  // the end of rows 0 and 2 to rows 1 and 3
  x += moved<0x143, 0xc>(x);  // the end of row 1 to rows 2 and 3
  return x;
}
__device__ __forceinline__ double of_lane(double x, int lane) {
  uint64_t const bits = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, lane) |
                                        (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), lane) << 32);
}
__device__ __forceinline__ double wave_sum(double x) { return of_lane(wave_upto(x), 63); }
__device__ __forceinline__ double load_shared(double const *p) {
  return __builtin_bit_cast(double, __hip_atomic_load((__attribute__((address_space(1))) uint64_t const *)(uint64_t const *)p,
                                                      __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ void store_shared(double *p, double x) {
  __hip_atomic_store((__attribute__((address_space(1))) uint64_t *)(uint64_t *)p, __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}

// ROUNDS: 16-byte pieces of a row that a lane holds of a strip.
template <class T, int ROUNDS>
__global__ __launch_bounds__(kThreads) void verify_drafts_kernel(VerifyParams const P) {
  constexpr int V = 16 / sizeof(T), kRound = 64 * V, kStrip = ROUNDS * kRound;
  typedef T piece __attribute__((ext_vector_type(V), aligned(alignof(T))));  // (rows begin anywhere)
  __shared__ int is_last;
  int const lane = threadIdx.x % 64, wave = threadIdx.x / 64, D = P.drafts, N = P.vocabulary;
  long long const b = blockIdx.y;
  T const *const target = static_cast<T const *>(P.target) + b * (D + 1) * N;
  T const *const draft = P.draft != nullptr ? static_cast<T const *>(P.draft) + b * D * N : nullptr;
  double const share_of = P.uniforms[b * (D + 1) + D];

  // how many drafts stay: a draft a lane
  int taken = D, refused_token = -1;
  for (int base = 0; base < D; base += 64) {
    int const i = base + lane;
    int x = -1;
    bool stays = i >= D;
    if (i < D) {
      double const u = P.uniforms[b * (D + 1) + i];
      x = P.tokens[b * D + i];
      if (x >= 0 && x < N) {
        double const p = static_cast<float>(target[(long long)i * N + x]);
        double const q = draft != nullptr ? static_cast<float>(draft[(long long)i * N + x]) : 1.0;
        stays = u * q < p;
      } else {
        x = -1;  // the end of the drafts, which refuses nothing
      }
    }
    uint64_t const ends = __ballot(!stays);
    if (ends != 0) {
      int const at = __builtin_ctzll(ends);
      taken = base + at;
      refused_token = __builtin_amdgcn_readlane(x, at);
      break;
    }
  }
  bool const refused = refused_token >= 0;
  T const *const p_row = target + (long long)taken * N, *const q_row = refused && draft != nullptr ? draft + (long long)taken * N : nullptr;
  int const without = refused && draft == nullptr ? refused_token : -1;

  // What a lane holds of a strip, all of it asked for before any is looked at: behind a test of its own each round's loads
  // would wait for the round before.  Zeros past the row's end.
  struct Held {
    piece p[ROUNDS], q[ROUNDS];
  };
  auto hold = [&](int strip, T const *of_q) {
    Held h;
    long long const base = (long long)strip * kStrip, j = base + lane * V;
    if (base + kStrip <= N) {
#pragma unroll
      for (int r = 0; r < ROUNDS; r++) {
        h.p[r] = *reinterpret_cast<piece const *>(p_row + j + r * kRound);
      }
      if (of_q != nullptr) {
#pragma unroll
        for (int r = 0; r < ROUNDS; r++) {
          h.q[r] = *reinterpret_cast<piece const *>(of_q + j + r * kRound);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < ROUNDS; r++) {
#pragma unroll
        for (int e = 0; e < V; e++) {
          long long const at = j + r * kRound + e;
          h.p[r][e] = at < N ? p_row[at] : static_cast<T>(0.0f);
          h.q[r][e] = at < N && of_q != nullptr ? of_q[at] : static_cast<T>(0.0f);
        }
      }
    }
    return h;
  };
  // The weights of its round r: what is left of the target's (less), and the target's own (all).  A NaN weighs nothing.
  auto weights = [&](Held const &h, int r, bool of_q, int skip, double (&less)[V], double (&all)[V]) {
#pragma unroll
    for (int e = 0; e < V; e++) {
      double const w = static_cast<float>(h.p[r][e]), l = of_q ? w - static_cast<double>(static_cast<float>(h.q[r][e])) : w;
      all[e] = w > 0.0 ? w : 0.0;
      less[e] = l > 0.0 && r * kRound + e != skip ? l : 0.0;
    }
  };
  // the place of the token that is left out among this lane's of a strip
  auto place_in = [&](int strip) {
    long long const at = without - (long long)strip * kStrip - lane * V;
    return without >= 0 && at >= 0 && at < kStrip ? (int)at : -1;
  };

  // this wavefront's strips, the next on its way while one is added up
  double *const parts = P.parts + 2 * b * P.strips;
  int const first_strip = ((int)blockIdx.x * kWaves + wave) * P.each;
  int const end_strip = first_strip + P.each < P.strips ? first_strip + P.each : P.strips;
  if (first_strip < end_strip) {
    Held next = hold(first_strip, q_row);
    for (int strip = first_strip; strip < end_strip; strip++) {
      Held const h = next;
      if (strip + 1 < end_strip) {
        next = hold(strip + 1, q_row);
      }
      int const skip = place_in(strip);
      double less_sum = 0.0, all_sum = 0.0;
#pragma unroll
      for (int r = 0; r < ROUNDS; r++) {
        double less[V], all[V];
        weights(h, r, q_row != nullptr, skip, less, all);
#pragma unroll
        for (int e = 0; e < V; e++) {
          less_sum += less[e];
          all_sum += all[e];
        }
      }
      less_sum = wave_sum(less_sum);
      all_sum = wave_sum(all_sum);
      if (lane < 2) {
        store_shared(parts + 2 * strip + lane, lane == 0 ? less_sum : all_sum);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    int const count = gridDim.x;
    is_last = 1;
    if (count > 1) {
      int *const ticket = P.tickets + b * State::kJoinStep;
      int const others = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      is_last = others == count - 1;
      if (others == count - 1) {
        __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
      }
    }
  }
  __syncthreads();
  if (is_last == 0 || wave != 0) {
    return;
  }

  // the totals, and the strip in which the sum passes the share (none: the last with a weight)
  double total[2] = {0.0, 0.0}, first_parts[2] = {0.0, 0.0};
  for (int i = lane; i < P.strips; i += 64) {
    double const its[2] = {load_shared(parts + 2 * i), load_shared(parts + 2 * i + 1)};
    first_parts[0] = i < 64 ? its[0] : first_parts[0];
    first_parts[1] = i < 64 ? its[1] : first_parts[1];
    total[0] += its[0];
    total[1] += its[1];
  }
  total[0] = wave_sum(total[0]);
  total[1] = wave_sum(total[1]);
  int const which = total[0] > 0.0 ? 0 : 1;
  double share = share_of * total[which], before = 0.0, upto_base = 0.0;
  int at_strip = -1, last_with = 0;
  for (int base = 0; base < P.strips && at_strip < 0; base += 64) {
    int const i = base + lane;
    double const its = base == 0 ? first_parts[which] : (i < P.strips ? load_shared(parts + 2 * i + which) : 0.0);
    double const upto = upto_base + wave_upto(its);
    uint64_t const passes = __ballot(its > 0.0 && upto > share), some = __ballot(its > 0.0);
    if (passes != 0) {
      int const at = __builtin_ctzll(passes);
      at_strip = base + at;
      before = of_lane(upto - its, at);
    } else if (some != 0) {
      last_with = base + 63 - __builtin_clzll(some);
    }
    upto_base = of_lane(upto, 63);
  }
  if (at_strip < 0) {
    at_strip = last_with;
    share = INFINITY;
  }

  // the token: the lanes of a round are in the order of their tokens
  int token = -1, last = -1;
  if (total[which] > 0.0) {
    T const *const of_q = which == 0 ? q_row : nullptr;
    Held const h = hold(at_strip, of_q);
    int const skip = which == 0 ? place_in(at_strip) : -1;
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
      double w[V], all[V], own = 0.0;
      weights(h, r, of_q != nullptr, skip, w, all);
#pragma unroll
      for (int e = 0; e < V; e++) {
        own += w[e];
      }
      double const through = wave_upto(own);
      double upto = before + (through - own);
      int const j = (int)((long long)at_strip * kStrip) + r * kRound + lane * V;
      int passing = -1, some = -1;
#pragma unroll
      for (int e = V - 1; e >= 0; e--) {
        some = some < 0 && w[e] > 0.0 ? j + e : some;
      }
#pragma unroll
      for (int e = 0; e < V; e++) {
        upto += w[e];
        passing = passing < 0 && w[e] > 0.0 && upto > share ? j + e : passing;
      }
      uint64_t const passes = __ballot(passing >= 0), any = __ballot(some >= 0);
      if (passes != 0 && token < 0) {
        token = __builtin_amdgcn_readlane(passing, __builtin_ctzll(passes));
      }
      if (any != 0) {
        last = __builtin_amdgcn_readlane(some, 63 - __builtin_clzll(any));
      }
      before += of_lane(through, 63);
    }
    token = token < 0 ? last : token;
  }
  for (int i = lane; i <= D; i += 64) {
    P.out[b * (D + 1) + i] = i < taken ? P.tokens[b * D + i] : (i == taken ? token : -1);
  }
  if (lane == 0) {
    P.accepted[b] = taken;
  }
}

template <class T, int ROUNDS>
int launch_rounds(VerifyParams P, int sequences, int most) {
  constexpr int kStrip = 64 * ROUNDS * (16 / (int)sizeof(T));
  P.strips = (P.vocabulary - 1) / kStrip + 1;
  P.each = 1;
  auto workgroups = [&]() { return (P.strips - 1) / (kWaves * P.each) + 1; };
  while (workgroups() > 1 && ((long long)sequences * workgroups() > most || sequences > State::kJoinWorkgroups)) {
    P.each = P.each < P.strips / 2 ? 2 * P.each : P.strips;
  }
  // as many sequences to a launch as the workspace has sums for, and a grid rows
  long long const fit = (long long)(state().scratch_bytes / (2 * sizeof(double))) / P.strips;
  int const slice = fit < 1 ? 0 : (int)(fit < 65535 ? fit : 65535);
  if (slice == 0) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_verify_drafts: a vocabulary of %d", P.vocabulary);
  }
  return in_slices(sequences, slice, [&](long long at, long long count) -> int {
    VerifyParams Q = P;
    Q.target = static_cast<T const *>(P.target) + at * (P.drafts + 1) * P.vocabulary;
    Q.draft = P.draft != nullptr ? static_cast<T const *>(P.draft) + at * P.drafts * P.vocabulary : nullptr;
    Q.tokens = P.tokens + at * P.drafts;
    Q.uniforms = P.uniforms + at * (P.drafts + 1);
    Q.accepted = P.accepted + at;
    Q.out = P.out + at * (P.drafts + 1);
    MI355_HIP(launch_kernel(verify_drafts_kernel<T, ROUNDS>, dim3((unsigned)workgroups(), (unsigned)count), dim3(kThreads), 0,
                            state().stream(), Q));
    return MI355_OK;
  });
}

// Strips of one round where all of them together are at most two workgroups a compute unit: the last workgroup then has
// one to look through.  Else four rounds, and as many of those to a wavefront as keep the workgroups to four a compute unit,
// one wave of them.  Measured (us, one round and four): 5.4 and 6.6 of 1 sequence x 32000 fp32, 5.8 and 9.0 of 19 x 50021 fp16.
template <class T>
int launch_verify(VerifyParams const &P, int sequences) {
  constexpr int kRound = kThreads * (16 / (int)sizeof(T));
  bool const few = (long long)sequences * ((P.vocabulary - 1) / kRound + 1) <= 512;
  return few ? launch_rounds<T, 1>(P, sequences, 512) : launch_rounds<T, 4>(P, sequences, 1024);
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355_verify_drafts(void const *target, void const *draft, int const *tokens, float const *uniforms, int *accepted,
                                   int *out, int sequences, int drafts, int vocabulary, int type) {
  MI355_REQUIRE_INIT();
  if (sequences < 0 || drafts < 0 || drafts == INT_MAX || vocabulary < 1) {
    return fail(MI355_ERR_INVALID, "mi355_verify_drafts: %d sequences, %d drafts, a vocabulary of %d", sequences, drafts, vocabulary);
  }
  if (type != MI355_TYPE_F16 && type != MI355_TYPE_BF16 && type != MI355_TYPE_F32) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_verify_drafts: type %d", type);
  }
  if (drafts > INT_MAX / 2) {  // (a wavefront goes through them in steps of 64, counted by an int)
    return fail(MI355_ERR_UNSUPPORTED, "mi355_verify_drafts: %d drafts", drafts);
  }
  if (sequences == 0) {
    return MI355_OK;
  }
  if (target == nullptr || (tokens == nullptr && drafts > 0) || uniforms == nullptr || accepted == nullptr || out == nullptr) {
    return fail(MI355_ERR_INVALID, "mi355_verify_drafts: null pointer");
  }
  State &s = state();
  VerifyParams const P{target, draft, tokens, uniforms, accepted, out, static_cast<double *>(s.scratch()), s.queue_join_tickets(), drafts, vocabulary, 0, 0};
  return type == MI355_TYPE_F16    ? launch_verify<_Float16>(P, sequences)
         : type == MI355_TYPE_BF16 ? launch_verify<__bf16>(P, sequences)
                                   : launch_verify<float>(P, sequences);
}
