// Verification of drafted tokens against the target model's probabilities (speculative sampling).
//
// Drafted token x_i (i < n) with draft probability q_i(x_i) is taken while u_i q_i(x_i) < p_i(x_i), u_i given in [0, 1); a
// draft without probabilities counts as certain (q = 1 at its token, 0 elsewhere).  At the first refusal r one token is drawn
// from the residual max(p_r - q_r, 0), after n taken drafts from p_n: the smallest j whose running sum of weights exceeds
// u_n times their total.  The products of two inputs are exact in 64 bits and the sums are held there, so that the outcome does
// not depend on how the vocabulary is split.
// Parity: the reference has no speculative decoding.
#include "common.cuh"

namespace b200k {
namespace {

struct VerifyParams {
  int B, n, V;
  int64_t p_sb, p_sn, q_sb, q_sn;     // element strides of the probabilities: sequence, position
  int64_t t_sb, u_sb;                 // of tokens and random numbers: sequence
};

constexpr int kVerifyThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(int64_t* __restrict__ taken_out, int64_t* __restrict__ out,
                                                                       const T* __restrict__ target, const T* __restrict__ draft,
                                                                       const int64_t* __restrict__ tokens,
                                                                       const float* __restrict__ uniforms, const VerifyParams p) {
  __shared__ int s_first;
  __shared__ double s_sum[kVerifyThreads + 1];
  const int b = blockIdx.x;
  const int64_t* tok = tokens + b * p.t_sb;
  const float* u = uniforms + b * p.u_sb;
  if (threadIdx.x == 0) s_first = p.n;
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += kVerifyThreads) {
    const int64_t x = tok[i];
    bool take = x >= 0 && x < p.V;
    if (take) {
      const double px = (double)ToF<T>::to(target[b * p.p_sb + i * p.p_sn + x]);
      const double qx = draft ? (double)ToF<T>::to(draft[b * p.q_sb + i * p.q_sn + x]) : 1.0;
      take = (double)u[i] * qx < px;
    }
    if (!take) atomicMin(&s_first, i);
  }
  __syncthreads();
  const int r = s_first;
  const T* prow = target + b * p.p_sb + r * p.p_sn;
  const int64_t x = r < p.n ? tok[r] : -1;
  const bool refused = x >= 0 && x < p.V;       // otherwise the draft ends here: the target's own distribution
  const T* qrow = refused && draft ? draft + b * p.q_sb + r * p.q_sn : nullptr;
  auto weight = [&](int j, bool residual) {
    double w = (double)ToF<T>::to(prow[j]);
    if (residual) {
      if (qrow) w -= (double)ToF<T>::to(qrow[j]);
      else if (j == x) w = 0.0;
    }
    return w > 0.0 ? w : 0.0;
  };
  const int per = (p.V + kVerifyThreads - 1) / kVerifyThreads, j0 = min(p.V, (int)threadIdx.x * per), j1 = min(p.V, j0 + per);
  int64_t token = -1;
  for (int round = refused ? 0 : 1; round < 2; ++round) {     // no residual left: the target's distribution
    double s = 0.0;
    for (int j = j0; j < j1; ++j) s += weight(j, round == 0);
    s_sum[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double run = 0.0;
      for (int t = 0; t < kVerifyThreads; ++t) { const double v = s_sum[t]; s_sum[t] = run; run += v; }
      s_sum[kVerifyThreads] = run;
    }
    __syncthreads();
    if (s_sum[kVerifyThreads] > 0.0) {
      if (threadIdx.x == 0) {
        const double limit = (double)u[p.n] * s_sum[kVerifyThreads];
        int seg = kVerifyThreads - 1;
        while (seg > 0 && s_sum[seg] > limit) --seg;
        double run = s_sum[seg];
        for (int j = seg * per; j < p.V; ++j) {
          const double w = weight(j, round == 0);
          run += w;
          if (w > 0.0) token = j;
          if (run > limit) break;
        }
      }
      break;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i <= p.n; i += kVerifyThreads)
    if (i != r) out[(int64_t)b * (p.n + 1) + i] = i < r ? tok[i] : -1;
  if (threadIdx.x == 0) {
    out[(int64_t)b * (p.n + 1) + r] = token;
    taken_out[b] = r;
  }
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int b200_verify_drafts(int dtype, int64_t* taken, int64_t* out, const void* target, const void* draft, const int64_t* tokens,
                                  const float* uniforms, int B, int n, int V, const int64_t* strides, cudaStream_t stream) {
  if (B <= 0 || n < 0 || V <= 0) return (int)cudaErrorNotSupported;
  const VerifyParams p{B, n, V, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5]};
  B200K_DISPATCH_FLOAT(dtype, T, {
    verify_drafts_kernel<T><<<B, kVerifyThreads, 0, stream>>>(taken, out, (const T*)target, (const T*)draft, tokens, uniforms, p);
  });
  B200K_LAUNCH_RET();
}
