// Rotary positions, and with them the write of new keys and values into a paged cache.
//
// A pair (a, b) of a head at position p becomes (a c - b s, b c + a s) with c = m cos(p w), s = m sin(p w).  p w is
// computed in 64 bits and reduced to a fraction of a turn before it is rounded: in 32 bits the angle of position 10^6
// would be 0.06 radians off.  The sines and cosines of a token are the same for all of its heads, so a workgroup
// computes them once, one pair a thread, into LDS.  Bound by the launch for a few tokens (3.9 us of 16), by HBM for many: 8192
// tokens with 32 + 8 heads of 128 move 201 MB in 40 us, the rate of a copy.
#include "common.h"

namespace mi355 {
namespace {

constexpr int kThreads = 256;
constexpr int kMostPairs = MI355_MAX_ROTARY_PAIRS;  // of a head: their sines and cosines are 8 KB of LDS

struct RotaryParams {
  void const *src[3];  // queries, keys, values
  long long src_stride[3];
  void *q_out, *k, *v;
  long long out_stride, page_stride, token_stride, head_stride;
  int const *positions, *slots;
  double const *angles;
  int tokens, q_heads, kv_heads, head_dim, pairs, page_size, slot_count, head_split;  // workgroups of a token
};

__device__ __forceinline__ float to_float(_Float16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_float(__bf16 x) { return static_cast<float>(x); }

// V elements moved at a time (1 or 8).  A unit of work is V pairs of a head, or V elements that are copied.
template <class T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryParams const P) {
  typedef T vec __attribute__((ext_vector_type(V)));
  __shared__ float2 turn[kMostPairs];
  int const token = blockIdx.x;
  double const position = P.positions[token];
  for (int i = threadIdx.x; i < P.pairs; i += kThreads) {
    double turns = position * P.angles[i] * 0.15915494309189533577;  // 1 / 2 pi
    turns -= __builtin_rint(turns);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns), &s, &c);
    float const m = static_cast<float>(P.angles[P.pairs + i]);
    turn[i] = float2{m * c, m * s};
  }
  int const slot = P.kv_heads != 0 ? P.slots[token] : -1;
  bool const kept = slot >= 0 && slot < P.slot_count;
  long long const cache_at =
      kept ? (long long)(slot / P.page_size) * P.page_stride + (long long)(slot % P.page_size) * P.token_stride : 0;
  __syncthreads();
  constexpr int W = INTERLEAVED && V > 1 ? V / 2 : V;  // pairs of a unit
  int const turned_units = P.pairs / W, units = turned_units + (P.head_dim - 2 * P.pairs) / V, whole = P.head_dim / V;
  int const q_all = P.q_heads * units, k_all = P.kv_heads * units, all = q_all + k_all + P.kv_heads * whole;
  for (int u = blockIdx.y * kThreads + threadIdx.x; u < all; u += kThreads * P.head_split) {
    int const which = u < q_all ? 0 : (u < q_all + k_all ? 1 : 2);
    int const local = which == 0 ? u : (which == 1 ? u - q_all : u - q_all - k_all), per = which == 2 ? whole : units;
    int const head = local / per, unit = local % per;
    if (which != 0 && !kept) {
      continue;
    }
    T const *const in = static_cast<T const *>(P.src[which]) + token * P.src_stride[which] + head * P.head_dim;
    T *const out = which == 0 ? static_cast<T *>(P.q_out) + token * P.out_stride + head * P.head_dim
                              : static_cast<T *>(which == 1 ? P.k : P.v) + cache_at + head * P.head_stride;
    if (which == 2 || unit >= turned_units) {
      int const e = which == 2 ? unit * V : 2 * P.pairs + (unit - turned_units) * V;
      *reinterpret_cast<vec *>(out + e) = *reinterpret_cast<vec const *>(in + e);
    } else if (INTERLEAVED && V > 1) {
      vec x = *reinterpret_cast<vec const *>(in + unit * V);
#pragma unroll
      for (int j = 0; j < V / 2; j++) {
        float2 const t = turn[unit * W + j];
        float const a = to_float(x[2 * j]), b = to_float(x[2 * j + 1]);
        x[2 * j] = static_cast<T>(a * t.x - b * t.y);
        x[2 * j + 1] = static_cast<T>(b * t.x + a * t.y);
      }
      *reinterpret_cast<vec *>(out + unit * V) = x;
    } else {
      int const first = INTERLEAVED ? 2 * unit : unit * V, second = INTERLEAVED ? first + 1 : first + P.pairs;
      vec x = *reinterpret_cast<vec const *>(in + first), y = *reinterpret_cast<vec const *>(in + second);
#pragma unroll
      for (int j = 0; j < V; j++) {
        float2 const t = turn[unit * W + j];
        float const a = to_float(x[j]), b = to_float(y[j]);
        x[j] = static_cast<T>(a * t.x - b * t.y);
        y[j] = static_cast<T>(b * t.x + a * t.y);
      }
      *reinterpret_cast<vec *>(out + first) = x;
      *reinterpret_cast<vec *>(out + second) = y;
    }
  }
}

// 16 bytes at a time where rows, heads and the pairs' runs begin at multiples of 16 bytes, else one element
bool wide(RotaryParams const &P, bool interleaved) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(P.q_out);
  long long strides = P.out_stride | P.head_dim | (interleaved ? 2 * P.pairs : P.pairs);
  for (int i = 0; i < (P.kv_heads != 0 ? 3 : 1); i++) {
    bits |= reinterpret_cast<uintptr_t>(P.src[i]);
    strides |= P.src_stride[i];
  }
  if (P.kv_heads != 0) {
    bits |= reinterpret_cast<uintptr_t>(P.k) | reinterpret_cast<uintptr_t>(P.v);
    strides |= P.page_stride | P.token_stride | P.head_stride;
  }
  return bits % 16 == 0 && strides % 8 == 0;
}

// A token's heads by as many workgroups as give each thread one unit of work, up to 1024 of them: measured (us, one workgroup
// and this) 4.3 and 3.9 of 16 tokens with 32 + 8 heads of 128, 5.7 and 3.9 of one with 128 + 16, 5.3 and 4.5 of 256 with
// 64 + 8.  Past that each computes the sines again for nothing: 40.2 of 8192 tokens would be 42.2 by two a token.
template <class T>
int launch_rotary(RotaryParams P, bool interleaved) {
  bool const by_eight = wide(P, interleaved);
  long long const units = (long long)(P.q_heads + P.kv_heads) * (P.head_dim - (interleaved && by_eight ? 0 : P.pairs)) + (long long)P.kv_heads * P.head_dim;
  long long const each = kThreads * (by_eight ? 8 : 1), most = P.tokens < 1024 ? 1024 / P.tokens : 1;
  P.head_split = (int)((units + each - 1) / each < most ? (units + each - 1) / each : most);
  auto *fn = by_eight ? (interleaved ? rotary_kernel<T, 8, true> : rotary_kernel<T, 8, false>)
                                  : (interleaved ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>);
  constexpr int kMostTokens = 1 << 23;  // of a launch, which has less than 2^32 threads
  for (int at = 0; at < P.tokens; at += kMostTokens) {
    RotaryParams Q = P;
    for (int i = 0; i < 3; i++) {
      Q.src[i] = static_cast<T const *>(P.src[i]) + at * P.src_stride[i];
    }
    Q.q_out = static_cast<T *>(P.q_out) + at * P.out_stride;
    Q.positions = P.positions + at;
    Q.slots = P.slots != nullptr ? P.slots + at : nullptr;
    int const count = P.tokens - at < kMostTokens ? P.tokens - at : kMostTokens;
    MI355_HIP(launch_kernel(fn, dim3((unsigned)count, (unsigned)P.head_split), dim3(kThreads), 0, state().stream(), Q));
    if (count < kMostTokens) {
      break;
    }
  }
  return MI355_OK;
}

int rotary(RotaryParams const &P, int interleaved, int type) {
  if (P.tokens < 0 || P.q_heads < 1 || P.head_dim < 1 || P.pairs < 1 || P.pairs > P.head_dim / 2) {
    return fail(MI355_ERR_INVALID, "rotary: %d tokens, %d heads of %d, %d pairs", P.tokens, P.q_heads, P.head_dim, P.pairs);
  }
  if (P.pairs > kMostPairs || (long long)(P.q_heads + 2LL * P.kv_heads) * P.head_dim > (1 << 30)) {
    return fail(MI355_ERR_UNSUPPORTED, "rotary: %d pairs of a head, or too many heads", P.pairs);
  }
  if (P.src_stride[0] < 0 || P.src_stride[1] < 0 || P.src_stride[2] < 0 || P.out_stride < 0 ||
      (P.tokens > 1 && P.out_stride < (long long)P.q_heads * P.head_dim)) {
    return fail(MI355_ERR_INVALID, "rotary: a stride below zero, or results of %d heads of %d that lie %lld apart", P.q_heads, P.head_dim,
                P.out_stride);
  }
  if (P.src[0] == P.q_out && P.src_stride[0] != P.out_stride && P.tokens > 1) {  // a token's results would lie on another's queries
    return fail(MI355_ERR_INVALID, "rotary: in place the strides are the same, not %lld and %lld", P.src_stride[0], P.out_stride);
  }
  if (type != MI355_TYPE_F16 && type != MI355_TYPE_BF16) {
    return fail(MI355_ERR_UNSUPPORTED, "rotary: type %d", type);
  }
  if (P.tokens == 0) {
    return MI355_OK;
  }
  if (P.src[0] == nullptr || P.q_out == nullptr || P.positions == nullptr || P.angles == nullptr) {
    return fail(MI355_ERR_INVALID, "rotary: null pointer");
  }
  return type == MI355_TYPE_F16 ? launch_rotary<_Float16>(P, interleaved != 0) : launch_rotary<__bf16>(P, interleaved != 0);
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355_rotary(void const *x, long long x_stride, void *y, long long y_stride, int const *positions,
                            double const *angles, int tokens, int heads, int head_dim, int pairs, int interleaved, int type) {
  MI355_REQUIRE_INIT();
  RotaryParams P{};
  P.src[0] = x;
  P.src_stride[0] = x_stride;
  P.q_out = y;
  P.out_stride = y_stride;
  P.positions = positions;
  P.angles = angles;
  P.tokens = tokens;
  P.q_heads = heads;
  P.head_dim = head_dim;
  P.pairs = pairs;
  return rotary(P, interleaved, type);
}

extern "C" int mi355_rotary_append(void const *q, long long q_stride, void const *k, long long k_stride, void const *v,
                                   long long v_stride, void *q_out, long long out_stride, int const *positions,
                                   double const *angles, int const *slots, mi355_paged_cache const *cache, int tokens, int q_heads,
                                   int pairs, int interleaved) {
  MI355_REQUIRE_INIT();
  if (cache == nullptr) {
    return fail(MI355_ERR_INVALID, "mi355_rotary_append: null cache");
  }
  if (int rc = check_paged_cache(*cache)) {
    return rc;
  }
  if (tokens > 0 && (k == nullptr || v == nullptr || slots == nullptr)) {
    return fail(MI355_ERR_INVALID, "mi355_rotary_append: null pointer");
  }
  RotaryParams P{};
  P.src[0] = q;
  P.src[1] = k;
  P.src[2] = v;
  P.src_stride[0] = q_stride;
  P.src_stride[1] = k_stride;
  P.src_stride[2] = v_stride;
  P.q_out = q_out;
  P.k = cache->k;
  P.v = cache->v;
  P.out_stride = out_stride;
  P.page_stride = cache->page_stride;
  P.token_stride = cache->token_stride;
  P.head_stride = cache->head_stride;
  P.positions = positions;
  P.slots = slots;
  P.angles = angles;
  P.tokens = tokens;
  P.q_heads = q_heads;
  P.kv_heads = cache->kv_heads;
  P.head_dim = cache->head_dim;
  P.pairs = pairs;
  P.page_size = cache->page_size;
  P.slot_count = cache->pages * cache->page_size;
  return rotary(P, interleaved, cache->type);
}
