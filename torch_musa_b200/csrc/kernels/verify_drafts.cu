// Verification of drafted tokens against the target model's probabilities (speculative sampling).
//
// Drafted token x_i (i < n) with draft probability q_i(x_i) is taken while u_i q_i(x_i) < p_i(x_i), u_i given in [0, 1); a
// draft without probabilities counts as certain (q = 1 at its token, 0 elsewhere).  At the first refusal r one token is drawn
// from the residual max(p_r - q_r, 0), after n taken drafts from p_n: the smallest j whose running sum of weights exceeds
// u_n times their total (u_n below zero or NaN counts as zero; from one on, the last j with a weight).  Products of two inputs are
// exact in 64 bits and the sums are held there.  Their order follows the split of the vocabulary, so the outcome depends on it where
// the limit lies within the sums' rounding, 2^-53 of the total for each addition, of a running sum.
//
// One cluster per sequence.  Every CTA of it finds r by itself (n small loads) and adds up its contiguous share of the row, a
// contiguous piece per warp; the pieces' sums cross the cluster through distributed shared memory, and the one warp in whose piece
// the limit falls goes over that piece again (it is in the L2 cache) with a running sum over its lanes.  So the row is read once
// from memory, in as many pieces as there are warps in the cluster.
// Parity: the reference has no speculative decoding.
#include "common.cuh"

namespace b200k {
namespace {

struct VerifyParams {
  int B, n, V;
  int split;                          // CTAs of a cluster
  int64_t p_sb, p_sn, q_sb, q_sn;     // element strides of the probabilities: sequence, position
  int64_t t_sb, u_sb;                 // of tokens and random numbers: sequence
};

constexpr int kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxPieces = 16 * kVerifyWarps;

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) v += __shfl_xor_sync(0xffffffffu, v, w);
  return v;
}

// kVec: rows start on 16 bytes, so four lanes' worth of a piece is loaded at a time
template <typename T, bool kVec>
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(int64_t* __restrict__ taken_out, int64_t* __restrict__ out,
                                                                       const T* __restrict__ target, const T* __restrict__ draft,
                                                                       const int64_t* __restrict__ tokens,
                                                                       const float* __restrict__ uniforms, const VerifyParams p) {
  constexpr int kN = kVec ? Vec16<T>::N : 1, kStep = 32 * kN;      // elements of a lane and of a warp per load
  __shared__ int s_first;
  __shared__ double s_mine[kVerifyWarps], s_all[kMaxPieces];
  const int b = blockIdx.x / p.split, rank = blockIdx.x - b * p.split, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  const double un = u[p.n] > 0.f ? (double)u[p.n] : 0.0;       // below zero or NaN: zero, so that some piece always has the limit
  // this warp's piece of the row, a whole number of its loads long
  const int pieces = p.split * kVerifyWarps, piece = rank * kVerifyWarps + warp;
  const int per = ((p.V + pieces - 1) / pieces + kStep - 1) / kStep * kStep;
  const int j0 = (int)min((int64_t)p.V, (int64_t)piece * per), j1 = (int)min((int64_t)p.V, (int64_t)j0 + per);
  auto load = [&](const T* row, int j, float (&v)[kN]) {
    if (kVec && j + kN <= p.V) {
      const Vec16<T> w = ld16(row + j);
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = ToF<T>::to(w.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = j + e < p.V ? ToF<T>::to(row[j + e]) : 0.f;
    }
  };
  // the weights of elements [j, j + kN): the residual, or the target's own
  auto weights = [&](int j, bool residual, double (&w)[kN]) {
    float pv[kN], qv[kN];
    load(prow, j, pv);
    if (residual && qrow) load(qrow, j, qv);
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      w[e] = (double)pv[e];
      if (residual && qrow) w[e] -= (double)qv[e];
      if (residual && !qrow && j + e == x) w[e] = 0.0;
      w[e] = w[e] > 0.0 ? w[e] : 0.0;          // NaN weighs nothing
    }
  };
  auto cluster_arrive = [&]() {
    if (p.split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  };
  auto cluster_wait = [&]() {
    if (p.split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
  };
  if (rank == 0)
    for (int i = threadIdx.x; i <= p.n; i += kVerifyThreads)
      if (i != r) out[(int64_t)b * (p.n + 1) + i] = i < r ? tok[i] : -1;
  for (int round = refused ? 0 : 1; round < 2; ++round) {     // no residual left: the target's distribution
    double s = 0.0;
#pragma unroll 4
    for (int j = j0 + lane * kN; j < j1; j += kStep) {
      double w[kN];
      weights(j, round == 0, w);
#pragma unroll
      for (int e = 0; e < kN; ++e) s += w[e];
    }
    s = warp_sum(s);
    if (lane == 0) s_mine[warp] = s;
    cluster_arrive();
    cluster_wait();
    for (int c = threadIdx.x; c < pieces; c += kVerifyThreads) {
      double v;
      if (p.split > 1) {
        uint32_t a = (uint32_t)__cvta_generic_to_shared(&s_mine[c % kVerifyWarps]);
        asm volatile("{\n\t.reg .u32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f64 %0, [r];\n\t}"
                     : "=d"(v) : "r"(a), "r"(c / kVerifyWarps) : "memory");
      } else {
        v = s_mine[c];
      }
      s_all[c] = v;
    }
    // a CTA leaves, or writes s_mine again, when all have read it: waited for at the end
    cluster_arrive();
    __syncthreads();
    // The running sum at the piece borders: one function of the border, evaluated the same way by both its neighbours, and it never
    // falls (sums of what is not negative, in a fixed order).  So exactly one warp finds the limit in its piece.
    double before = 0.0, upto = 0.0, total = 0.0;
    for (int c = lane; c < pieces; c += 32) {
      const double v = s_all[c];
      before += c < piece ? v : 0.0;
      upto += c <= piece ? v : 0.0;
      total += v;
    }
    before = warp_sum(before);
    upto = warp_sum(upto);
    total = warp_sum(total);
    if (total > 0.0) {
      const double limit = un * total;
      const bool here = limit < total ? before <= limit && limit < upto : before < total && upto == total;
      if (here) {
        double run = before;
        int token = -1;
        for (int j = j0; j < j1; j += kStep) {
          double w[kN], mine = 0.0;
          weights(j + lane * kN, round == 0, w);
#pragma unroll
          for (int e = 0; e < kN; ++e) mine += j + lane * kN + e < j1 ? w[e] : 0.0;
          double scan = mine;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, scan, d);
            if (lane >= d) scan += y;
          }
          double start = __shfl_up_sync(0xffffffffu, scan, 1);
          start = run + (lane > 0 ? start : 0.0);
          int found = -1, last = -1;
          double acc = start;
#pragma unroll
          for (int e = 0; e < kN; ++e) {
            if (j + lane * kN + e >= j1) continue;
            acc += w[e];
            if (w[e] > 0.0) last = j + lane * kN + e;
            if (found < 0 && w[e] > 0.0 && acc > limit) found = j + lane * kN + e;
          }
          const uint32_t any = __ballot_sync(0xffffffffu, found >= 0), weight = __ballot_sync(0xffffffffu, last >= 0);
          if (any) {
            token = __shfl_sync(0xffffffffu, found, __ffs(any) - 1);
            break;
          }
          if (weight) token = __shfl_sync(0xffffffffu, last, 31 - __clz(weight));     // stands if rounding leaves no later one
          run = __shfl_sync(0xffffffffu, run + scan, 31);
        }
        if (lane == 0) out[(int64_t)b * (p.n + 1) + r] = token;
      }
      if (rank == 0 && threadIdx.x == 0) taken_out[b] = r;
      __syncwarp();
      cluster_wait();
      return;
    }
    cluster_wait();
  }
  if (rank == 0 && threadIdx.x == 0) {
    out[(int64_t)b * (p.n + 1) + r] = -1;
    taken_out[b] = r;
  }
}

template <typename T>
int launch_verify(int64_t* taken, int64_t* out, const T* target, const T* draft, const int64_t* tokens, const float* uniforms, VerifyParams p,
                  cudaStream_t stream) {
  // CTAs of a cluster: as many as leave every thread a load or two, up to eight while there are places for all of them, sixteen only
  // where each gets an SM (four drafts, 32000 words, us in a graph for 2 / 4 / 8 / 16: one sequence 10.6 / 7.7 / 6.3 / 5.4; with seven
  // drafts 64 sequences 19.6 / 12.2 / 9.0 / 14.8)
  const int loads = (int)cdiv(p.V, (int64_t)kVerifyThreads * Vec16<T>::N);
  p.split = 1;
  while (p.split < 16 && p.split < loads && 2ll * p.B * p.split <= (p.split < 8 ? 4 : 1) * kSMs) p.split *= 2;
  if ((long long)p.B * p.split > 2147483647ll) return (int)cudaErrorNotSupported;
  auto on16 = [](const T* x, int64_t s0, int64_t s1) { return aligned16(x) && s0 % Vec16<T>::N == 0 && s1 % Vec16<T>::N == 0; };
  const bool vec = on16(target, p.p_sb, p.p_sn) && (!draft || on16(draft, p.q_sb, p.q_sn));
  static OncePerDevice once;
  if (int e = once([] {
        if (int r = (int)cudaFuncSetAttribute(verify_drafts_kernel<T, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return r;
        return (int)cudaFuncSetAttribute(verify_drafts_kernel<T, false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      }))
    return e;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)p.split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(p.B * p.split));
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = p.split > 1 ? 1 : 0;
  const cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, verify_drafts_kernel<T, true>, taken, out, target, draft, tokens, uniforms, p)
                            : cudaLaunchKernelEx(&cfg, verify_drafts_kernel<T, false>, taken, out, target, draft, tokens, uniforms, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return (int)e;
  }
  note_launch();
  return 0;
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int b200_verify_drafts(int dtype, int64_t* taken, int64_t* out, const void* target, const void* draft, const int64_t* tokens,
                                  const float* uniforms, int B, int n, int V, const int64_t* strides, cudaStream_t stream) {
  if (B <= 0 || n < 0 || V <= 0 || V > 2147483647 - 65536) return (int)cudaErrorNotSupported;
  const VerifyParams p{B, n, V, 1, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5]};
  B200K_DISPATCH_FLOAT(dtype, T, { return launch_verify<T>(taken, out, (const T*)target, (const T*)draft, tokens, uniforms, p, stream); });
  return (int)cudaErrorNotSupported;
}
