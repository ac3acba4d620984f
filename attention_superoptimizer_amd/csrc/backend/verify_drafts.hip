// Speculative sampling's decision about drafted tokens.
//
// Draft i stays while u_i q_i(x_i) < p_i(x_i): the product of two 24-bit numbers is exact in 64 bits.  The next token is
// the lowest j whose sum of weights w_0 + .. + w_j passes u times their total, summed in 64 bits: among 10^5 weights
// 32-bit sums would be off by whole tokens.
#include "common.h"

#include <climits>

namespace mi355 {
namespace {

constexpr int kThreads = 256;

struct VerifyParams {
  void const *target, *draft;
  int const *tokens;
  float const *uniforms;
  int *accepted, *out;
  int sequences, drafts, vocabulary;
};

// The weight of a token at the place after the drafts that were taken.  A NaN counts as nothing.
template <class T>
struct Weights {
  T const *target, *draft;  // the place's rows; draft null: no draft refused, or a certain one
  int without;              // the token of a certain draft that was refused, or -1
  __device__ __forceinline__ double operator()(int j) const {
    double w = static_cast<double>(static_cast<float>(target[j]));
    if (draft != nullptr) {
      w -= static_cast<double>(static_cast<float>(draft[j]));
    }
    return w > 0.0 && j != without ? w : 0.0;
  }
};

__device__ __forceinline__ double block_sum(double x, double *lds) {
  for (int off = 32; off > 0; off >>= 1) {
    x += __shfl_xor(x, off, 64);
  }
  __syncthreads();
  if (threadIdx.x % 64 == 0) {
    lds[threadIdx.x / 64] = x;
  }
  __syncthreads();
  double total = 0.0;
  for (int w = 0; w < kThreads / 64; w++) {
    total += lds[w];
  }
  return total;
}

// A workgroup per sequence: the total of the weights, then tiles of 256 from the first on until the sum passes.
template <class T>
__global__ __launch_bounds__(kThreads) void verify_drafts_kernel(VerifyParams const P) {
  __shared__ double parts[kThreads / 64], sums[kThreads];
  __shared__ int found, last;
  long long const b = blockIdx.x;
  int const V = P.vocabulary, D = P.drafts, tid = threadIdx.x;
  T const *const target = static_cast<T const *>(P.target) + b * (D + 1) * V;
  T const *const draft = P.draft != nullptr ? static_cast<T const *>(P.draft) + b * D * V : nullptr;
  int taken = 0;
  bool refused = false;
  while (taken < D) {
    int const x = P.tokens[b * D + taken];
    if (x < 0 || x >= V) {
      break;
    }
    double const p = static_cast<float>(target[(long long)taken * V + x]);
    double const q = draft != nullptr ? static_cast<float>(draft[(long long)taken * V + x]) : 1.0;
    if (!(static_cast<double>(P.uniforms[b * (D + 1) + taken]) * q < p)) {
      refused = true;
      break;
    }
    taken++;
  }
  Weights<T> w{target + (long long)taken * V, refused && draft != nullptr ? draft + (long long)taken * V : nullptr,
               refused && draft == nullptr ? P.tokens[b * D + taken] : -1};
  double total = 0.0;
  for (int pass = 0; pass < 2; pass++) {
    double mine = 0.0;
    for (int j = tid; j < V; j += kThreads) {
      mine += w(j);
    }
    total = block_sum(mine, parts);
    if (total > 0.0 || !refused) {
      break;
    }
    w.draft = nullptr;  // the differences are all zero
    w.without = -1;
  }
  if (tid == 0) {
    found = INT_MAX;
    last = -1;
  }
  __syncthreads();
  double const share = static_cast<double>(P.uniforms[b * (D + 1) + D]) * total;
  double before = 0.0;
  for (int base = 0; base < V && total > 0.0; base += kThreads) {
    int const j = base + tid;
    double const mine = j < V ? w(j) : 0.0;
    sums[tid] = mine;
    __syncthreads();
    double upto = before;
    for (int i = 0; i <= tid; i++) {
      upto += sums[i];
    }
    if (mine > 0.0) {
      atomicMax(&last, j);
      if (upto > share) {
        atomicMin(&found, j);
      }
    }
    double const whole = block_sum(mine, parts);
    before += whole;
    if (found != INT_MAX) {
      break;
    }
    __syncthreads();
  }
  __syncthreads();
  if (tid <= D) {
    int const token = found != INT_MAX ? found : last;
    P.out[b * (D + 1) + tid] = tid < taken ? P.tokens[b * D + tid] : (tid == taken ? token : -1);
  }
  for (int i = tid + kThreads; i <= D; i += kThreads) {
    int const token = found != INT_MAX ? found : last;
    P.out[b * (D + 1) + i] = i < taken ? P.tokens[b * D + i] : (i == taken ? token : -1);
  }
  if (tid == 0) {
    P.accepted[b] = taken;
  }
}

}  // namespace
}  // namespace mi355

using namespace mi355;

extern "C" int mi355_verify_drafts(void const *target, void const *draft, int const *tokens, float const *uniforms, int *accepted,
                                   int *out, int sequences, int drafts, int vocabulary, int type) {
  MI355_REQUIRE_INIT();
  if (sequences < 0 || drafts < 0 || vocabulary < 1) {
    return fail(MI355_ERR_INVALID, "mi355_verify_drafts: %d sequences, %d drafts, a vocabulary of %d", sequences, drafts, vocabulary);
  }
  if (type != MI355_TYPE_F16 && type != MI355_TYPE_BF16 && type != MI355_TYPE_F32) {
    return fail(MI355_ERR_UNSUPPORTED, "mi355_verify_drafts: type %d", type);
  }
  if (sequences == 0) {
    return MI355_OK;
  }
  if (target == nullptr || (tokens == nullptr && drafts > 0) || uniforms == nullptr || accepted == nullptr || out == nullptr) {
    return fail(MI355_ERR_INVALID, "mi355_verify_drafts: null pointer");
  }
  VerifyParams const P{target, draft, tokens, uniforms, accepted, out, sequences, drafts, vocabulary};
  auto *fn = type == MI355_TYPE_F16    ? verify_drafts_kernel<_Float16>
             : type == MI355_TYPE_BF16 ? verify_drafts_kernel<__bf16>
                                       : verify_drafts_kernel<float>;
  MI355_HIP(launch_kernel(fn, dim3((unsigned)sequences), dim3(kThreads), 0, state().stream(), P));
  return MI355_OK;
}
