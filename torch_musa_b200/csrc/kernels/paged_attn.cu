// Attention of the newest tokens of each sequence over a paged key-value cache, and the rotary embedding that writes it.
//
// The cache is a pool of pages [num_pages, Hkv, page_size, D] for keys and one for values; row b of the block table names
// the pages of sequence b in order.  seq_lens[b] counts the tokens of the sequence that are in the cache, the newest
// included, so token i of n new ones stands at position len - n + i.  Everything that changes from step to step is read
// on the device, so that a captured step can be replayed.
// Parity: the reference has no paged cache; its decoding goes through the vendor SDPA on contiguous keys (reference
// torch_musa/csrc/aten/ops/attention/mudnn/SDP.cpp).
#include "common.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <cstdlib>
#include <initializer_list>
#include <type_traits>

namespace cg = cooperative_groups;

namespace b200k {
namespace {

struct PagedParams {
  int B, n, H, Hkv;
  int num_pages, page_size, table_width;
  int page_shift;             // log2(page_size), or -1
  int window, sinks;          // window <= 0: every earlier key is visible
  int row_groups, split;      // CTAs of one (sequence, key head): row groups x shares of the keys
  float scale_log2;
  int64_t q_sb, q_sn, q_sh;                    // element strides; rows of D contiguous elements
  int64_t k_sp, k_sh, k_sr, v_sp, v_sh, v_sr;  // page, head, row in the page
  int64_t table_sb;
  const int* table;
  const int* lens;
  int* status;
};

constexpr int kPagedWarps = 4;
constexpr int kStepKeys = 16;          // keys of one step of a warp: they lie in one page
constexpr int kWarpRing = 16 * 1024;   // bytes of keys and values that a warp has in flight or in hand
constexpr int kMaxSplit = 16;          // CTAs of a cluster

template <int D> constexpr int ring_stages() { return kWarpRing / (kStepKeys * D * 2 * 2); }

__device__ __forceinline__ uint32_t shared_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes from global to shared memory without a register; zeros when `bytes` is 0
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// four 8 x 8 matrices of 16-bit values, one row address per lane; _t: transposed
__device__ __forceinline__ uint4 ldmatrix(uint32_t a) {
  uint4 r;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint4 ldmatrix_t(uint32_t a) {
  uint4 r;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (a, b) as 16-bit values, and what that rounding left of them
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  T h[2] = {ToF<T>::from(a), ToF<T>::from(b)}, l[2] = {ToF<T>::from(a - ToF<T>::to(h[0])), ToF<T>::from(b - ToF<T>::to(h[1]))};
  hi = *reinterpret_cast<const uint32_t*>(h);
  lo = *reinterpret_cast<const uint32_t*>(l);
}
// whether one of the two 16-bit values is infinite or NaN: its exponent bits are all set
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

// One CTA: one row group (up to 16 * MT rows = new tokens x query heads of a key head) of one (sequence, key head), one of C
// contiguous shares of the visible keys.  A share is cut into steps of 16 keys that the four warps take in turn; each warp runs its
// own online softmax, the warps join through shared memory and the C CTAs of a cluster through distributed shared memory.
//
// A warp copies the 16 rows of keys and of values of a step into a stage of its own ring (cp.async, whole rows at a time, 16-byte
// pieces swapped by row so that the eight rows of a matrix lie in different banks) and reads them as operands of mma m16n8k16:
//   S = Q K^T  (16 rows x 16 keys) with ldmatrix, O += P V (16 rows x D dimensions, 16 keys deep) with ldmatrix.trans.
// P is S's accumulator layout, and goes in as a 16-bit value plus the 16-bit remainder of its rounding (2^-16 or better).
template <typename T, int D, int MT>
__global__ void __launch_bounds__(kPagedWarps * 32, MT == 1 ? 3 : 2) paged_attn_kernel(T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ kp,
                                                                         const T* __restrict__ vp, const PagedParams p) {
  constexpr int kRows = 16 * MT, kStages = ring_stages<D>(), kStage = kStepKeys * D * 4;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_m[kPagedWarps][kRows], s_l[kPagedWarps][kRows];
  __shared__ float s_top[kRows], s_sum[kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.H / p.Hkv, rows_all = p.n * G;
  const int rank = (int)(blockIdx.x % p.split);
  int unit = (int)(blockIdx.x / p.split);
  const int group = unit % p.row_groups;
  unit /= p.row_groups;
  const int hk = unit % p.Hkv, b = unit / p.Hkv;
  const int r0 = group * kRows, rows = min(kRows, rows_all - r0);
  const int len = (int)min((long long)max(__ldg(p.lens + b), 0), (long long)p.table_width * p.page_size);
  // positions of the oldest and the newest token of the group; the steps of 16 keys that one of them sees
  const int pos0 = len - p.n + r0 / G, pos1 = len - p.n + (r0 + rows - 1) / G;
  const int wlo = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
  const int end = pos1 >= 0 ? pos1 / kStepKeys + 1 : 0;
  const int sink_steps = min(end, (p.sinks + kStepKeys - 1) / kStepKeys), first = max(wlo / kStepKeys, sink_steps);
  const int steps = sink_steps + max(0, end - first);
  const int s0 = (int)((long long)steps * rank / p.split), s1 = (int)((long long)steps * (rank + 1) / p.split);
  auto key_of = [&](int s) { return (s < sink_steps ? s : s - sink_steps + first) * kStepKeys; };

  // Q as operands: rows g and g + 8 of each 16, dimensions 16 ks + 2 t and 8 further
  uint4 qf[D / 16];
  uint4* sq = reinterpret_cast<uint4*>(smem + kPagedWarps * kWarpRing) + lane;      // MT == 2: [m][ks][lane], they would not fit
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (MT > 1 && warp != m) continue;
    const T* row[2];
    bool real[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = m * 16 + half * 8 + g;
      real[half] = r < rows;
      row[half] = q + b * p.q_sb + (r0 + r) / G * p.q_sn + (hk * G + (r0 + r) % G) * p.q_sh + 2 * t;
    }
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      auto word = [&](int half, int d) { return real[half] ? __ldg(reinterpret_cast<const uint32_t*>(row[half] + d)) : 0u; };
      const uint4 x = make_uint4(word(0, ks * 16), word(1, ks * 16), word(0, ks * 16 + 8), word(1, ks * 16 + 8));
      if constexpr (MT == 1) qf[ks] = x;
      else sq[(m * (D / 16) + ks) * 32] = x;
    }
  }

  const uint32_t ring = shared_u32(smem) + warp * kWarpRing;
  const int* table = p.table + b * p.table_sb;
  constexpr int kPieces = D / 8, kPerCopy = 32 / kPieces;      // 16-byte pieces of a row, rows that one instruction copies
  const int crow = lane / kPieces, cpiece = lane % kPieces;
  const T* kbase = kp + hk * p.k_sh + crow * p.k_sr + cpiece * 8;
  const T* vbase = vp + hk * p.v_sh + crow * p.v_sr + cpiece * 8;
  const int mi = lane >> 3, mr = lane & 7;
  // a lane's row address in a stage for ldmatrix; the piece 2 x of a row is at ((2 x) ^ swap) * 16, for x < 4
  const uint32_t krow = (uint32_t)(((mi >> 1) * 8 + mr) * D * 2), kswap = (uint32_t)(((mi & 1) ^ mr) * 16);
  const uint32_t vrow = (uint32_t)(kStepKeys * D * 2 + ((mi & 1) * 8 + mr) * D * 2), vswap = (uint32_t)(((mi >> 1) ^ mr) * 16);
  auto entry = [&](int s) {          // the page number of a step, read one step before it is needed
    if (s >= s1) return -1;
    const int k0 = key_of(s);
    return __ldg(table + (p.page_shift >= 0 ? k0 >> p.page_shift : k0 / p.page_size));
  };
  uint32_t found = 0;                // one bit a stage: whether the page of its step is in the pool
  auto issue = [&](int s, int number, int stage) {
    if (s < s1) {
      const int k0 = key_of(s);
      const bool there = number >= 0 && number < p.num_pages;
      if (!there && lane == 0 && p.status) atomicExch(p.status, 1);
      found = (found & ~(1u << stage)) | ((uint32_t)there << stage);
      const int64_t row = p.page_shift >= 0 ? k0 & (p.page_size - 1) : k0 % p.page_size, page = there ? number : 0;
      const T* ks = kbase + page * p.k_sp + row * p.k_sr;
      const T* vs = vbase + page * p.v_sp + row * p.v_sr;
      const uint32_t dst = ring + stage * kStage + (uint32_t)(crow * D * 2);
      // keys that no row sees are not read: zeros instead (with a probability of zero nothing else would be safe)
      auto copy = [&](auto whole) {
#pragma unroll
        for (int i = 0; i < kStepKeys / kPerCopy; ++i) {
          const int r = i * kPerCopy + crow, j = k0 + r;
          const int n16 = decltype(whole)::value || (there && j <= pos1 && (j >= wlo || j < p.sinks)) ? 16 : 0;
          const uint32_t d = dst + (uint32_t)(i * kPerCopy * D * 2) + (uint32_t)((cpiece ^ (r & 7)) * 16);
          copy16(d, ks + i * kPerCopy * p.k_sr, n16);
          copy16(d + kStepKeys * D * 2, vs + i * kPerCopy * p.v_sr, n16);
        }
      };
      if (there && k0 + kStepKeys - 1 <= pos1 && (k0 >= wlo || k0 + kStepKeys <= p.sinks)) copy(std::true_type{});
      else copy(std::false_type{});
    }
    copy_commit();
  };

  float o[MT][D / 8][4], m_run[MT][2], l_run[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int x = 0; x < D / 8; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][x][e] = 0.f;
    m_run[m][0] = m_run[m][1] = -INFINITY;
    l_run[m][0] = l_run[m][1] = 0.f;
  }

  if constexpr (MT > 1) __syncthreads();
  int s = s0 + warp, fetch = s;
  int number = entry(fetch);
#pragma unroll
  for (int st = 0; st < kStages; ++st) {
    const int now = number;
    number = entry(fetch + kPagedWarps);
    issue(fetch, now, st);
    fetch += kPagedWarps;
  }
  int stage = 0;
  for (; s < s1; s += kPagedWarps) {
    copy_wait<kStages - 1>();
    __syncwarp();
    const int k0 = key_of(s);
    const uint32_t src = ring + stage * kStage;
    float sc[MT][2][4];
    {
      float part[MT][2][4];          // odd products: four chains of half the length instead of two
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[m][nt][e] = part[m][nt][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint4 kf = ldmatrix(src + krow + (((uint32_t)(ks & 3) * 32) ^ kswap) + (uint32_t)(ks >> 2) * 128);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 x = MT == 1 ? qf[ks] : sq[(m * (D / 16) + ks) * 32];
          const uint32_t a[4] = {x.x, x.y, x.z, x.w};
          mma16816<T>(ks & 1 ? part[m][0] : sc[m][0], a, kf.x, kf.y);
          mma16816<T>(ks & 1 ? part[m][1] : sc[m][1], a, kf.z, kf.w);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[m][nt][e] += part[m][nt][e];
    }
    auto values = [&](int j) {         // the operands of dimensions [8 j, 8 j + 16), j even
      return ldmatrix_t(src + vrow + (((uint32_t)(j & 7) * 16) ^ vswap) + (uint32_t)(j >> 3) * 128);
    };
    const bool there = (found >> stage) & 1u;
    const bool all = there && k0 + kStepKeys - 1 <= pos0 && (p.window <= 0 || k0 > pos1 - p.window || k0 + kStepKeys <= p.sinks);
    const bool mixed = !all && pos0 != pos1;
    auto sees = [&](int pos, int j) { return there && j <= pos && (p.window <= 0 || j > pos - p.window || j < p.sinks); };

#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float mx[2];
      if (!all) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int pos = len - p.n + (r0 + m * 16 + half * 8 + g) / G;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!sees(pos, k0 + nt * 8 + 2 * t + e)) sc[m][nt][half * 2 + e] = -INFINITY;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x = fmaxf(fmaxf(sc[m][0][half * 2], sc[m][0][half * 2 + 1]), fmaxf(sc[m][1][half * 2], sc[m][1][half * 2 + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        mx[half] = x * p.scale_log2;
      }
      if (__any_sync(0xffffffffu, mx[0] > m_run[m][0] || mx[1] > m_run[m][1])) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float m_new = fmaxf(m_run[m][half], mx[half]);
          const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m_run[m][half] - m_new);
          m_run[m][half] = m_new;
          l_run[m][half] *= alpha;
#pragma unroll
          for (int x = 0; x < D / 8; ++x) {
            o[m][x][half * 2] *= alpha;
            o[m][x][half * 2 + 1] *= alpha;
          }
        }
      }
      uint32_t hi[4], lo[4];      // rows g and g + 8 of keys 2t.., then of keys 2t + 8..
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float ref = m_run[m][half] == -INFINITY ? 0.f : m_run[m][half];
          const float p0 = exp2_fast(fmaf(sc[m][nt][half * 2], p.scale_log2, -ref)), p1 = exp2_fast(fmaf(sc[m][nt][half * 2 + 1], p.scale_log2, -ref));
          l_run[m][half] += p0 + p1;
          split2<T>(p0, p1, hi[nt * 2 + half], lo[nt * 2 + half]);
        }
      bool careful = false;
      if (mixed) {
        bool odd = false;
#pragma unroll 1
        for (int j = 0; j < D / 8; j += 2) {
          const uint4 v = values(j);
          odd = odd || not_finite<T>(v.x) || not_finite<T>(v.y) || not_finite<T>(v.z) || not_finite<T>(v.w);
        }
        careful = __any_sync(0xffffffffu, odd);
      }
      if (!careful) {
#pragma unroll
        for (int j = 0; j < D / 8; j += 2) {
          const uint4 v = values(j);
          mma16816<T>(o[m][j], hi, v.x, v.y);
          mma16816<T>(o[m][j + 1], hi, v.z, v.w);
          mma16816<T>(o[m][j], lo, v.x, v.y);
          mma16816<T>(o[m][j + 1], lo, v.z, v.w);
        }
      } else {
        // An infinity or a NaN among values that some rows see and others do not: token by token, with the values that the token
        // does not see as zeros, and only its own rows kept.
        for (int pos = pos0; pos <= pos1; ++pos) {
          const uint32_t see0 = (sees(pos, k0 + 2 * t) ? 0xffffu : 0u) | (sees(pos, k0 + 2 * t + 1) ? 0xffff0000u : 0u);
          const uint32_t see1 = (sees(pos, k0 + 2 * t + 8) ? 0xffffu : 0u) | (sees(pos, k0 + 2 * t + 9) ? 0xffff0000u : 0u);
          const bool mine = len - p.n + (r0 + m * 16 + g) / G == pos, mine8 = len - p.n + (r0 + m * 16 + 8 + g) / G == pos;
#pragma unroll
          for (int j = 0; j < D / 8; j += 2) {
            const uint4 v = values(j);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816<T>(acc, hi, (x ? v.z : v.x) & see0, (x ? v.w : v.y) & see1);
              mma16816<T>(acc, lo, (x ? v.z : v.x) & see0, (x ? v.w : v.y) & see1);
              if (mine) { o[m][j + x][0] += acc[0]; o[m][j + x][1] += acc[1]; }
              if (mine8) { o[m][j + x][2] += acc[2]; o[m][j + x][3] += acc[3]; }
            }
          }
        }
      }
    }
    __syncwarp();
    const int now = number;
    number = entry(fetch + kPagedWarps);
    issue(fetch, now, stage);
    fetch += kPagedWarps;
    if (++stage == kStages) stage = 0;
  }

  // ---- the warps' parts: maxima and sums first, then the outputs relative to the common maximum
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float l = l_run[m][half];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t == 0) {
        s_m[warp][m * 16 + half * 8 + g] = m_run[m][half];
        s_l[warp][m * 16 + half * 8 + g] = l;
      }
    }
  copy_wait<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);            // [warps][kRows][D]
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = m * 16 + half * 8 + g;
      float top = s_m[0][r];
#pragma unroll
      for (int w = 1; w < kPagedWarps; ++w) top = fmaxf(top, s_m[w][r]);
      const float f = m_run[m][half] == -INFINITY ? 1.f : exp2_fast(m_run[m][half] - top);   // no key: zeros, or NaN
      if (warp == 0 && t == 0) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) {
          const float lw = s_l[w][r];
          sum += s_m[w][r] == -INFINITY ? lw : lw * exp2_fast(s_m[w][r] - top);
        }
        s_top[r] = top;
        s_sum[r] = sum;
      }
      float* dst = part + ((size_t)warp * kRows + r) * D + 2 * t;
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(dst + j * 8) = make_float2(o[m][j][half * 2] * f, o[m][j][half * 2 + 1] * f);
    }
  __syncthreads();
  auto store = [&](int r, int d, const float (&v)[4], float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;       // no key: zeros
    T o4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o4[e] = ToF<T>::from(sum == 0.f ? 0.f : v[e] * inv);
    const int i = (r0 + r) / G, h = hk * G + (r0 + r) % G;
    *reinterpret_cast<uint2*>(out + (((int64_t)b * p.n + i) * p.H + h) * D + d) = *reinterpret_cast<const uint2*>(o4);
  };
  if (p.split == 1) {
    for (int x = threadIdx.x * 4; x < rows * D; x += kPagedWarps * 32 * 4) {
      float v[4] = {};
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(part + w * kRows * D + x);
        v[0] += y.x; v[1] += y.y; v[2] += y.z; v[3] += y.w;
      }
      store(x / D, x % D, v, s_sum[x / D]);
    }
    return;
  }
  for (int x = threadIdx.x * 4; x < rows * D; x += kPagedWarps * 32 * 4) {       // the CTA's sum, over warp 0's part
    float4 v = *reinterpret_cast<const float4*>(part + x);
#pragma unroll
    for (int w = 1; w < kPagedWarps; ++w) {
      const float4 y = *reinterpret_cast<const float4*>(part + w * kRows * D + x);
      v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
    }
    *reinterpret_cast<float4*>(part + x) = v;
  }
  // ---- the cluster's parts: every CTA finishes its share of the elements
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int quads = rows * D / 4, share = (quads + p.split - 1) / p.split;
  for (int x = rank * share + threadIdx.x; x < min(quads, (rank + 1) * share); x += kPagedWarps * 32) {
    const int r = x * 4 / D;
    float top = -INFINITY, sum = 0.f, v[4] = {};
    for (int c = 0; c < p.split; ++c) top = fmaxf(top, *cluster.map_shared_rank(&s_top[r], c));
    for (int c = 0; c < p.split; ++c) {
      const float mc = *cluster.map_shared_rank(&s_top[r], c), lc = *cluster.map_shared_rank(&s_sum[r], c);
      const float4 y = *cluster.map_shared_rank(reinterpret_cast<const float4*>(part) + x, c);
      const float f = mc == -INFINITY ? 1.f : exp2_fast(mc - top);      // a CTA without a key has zeros
      sum += lc * f;
      v[0] += y.x * f; v[1] += y.y * f; v[2] += y.z * f; v[3] += y.w * f;
    }
    store(r, x * 4 % D, v, sum);
  }
  cluster.sync();
}

struct PagedWriteParams {
  int T, B, H, Hkv, D;
  int num_pages, page_size, table_width, table_len;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;     // of the inputs: token, head
  int64_t kp_sp, kp_sh, kp_sr, vp_sp, vp_sh, vp_sr;
  int64_t table_sb;
  const float* cosv;
  const float* sinv;
  const int* table;
  const int* lens;
  const int* cu;      // NULL: every sequence has T / B tokens
  int* status;
};

// q_out = rotate(q); rotate(k) and v go to their rows of the cache.  A thread owns eight adjacent dimensions of the first half
// of a row and their partners in the second half: two 16-byte loads and stores.
template <typename T>
__global__ void __launch_bounds__(256) paged_rope_kernel(T* __restrict__ q_out, const T* __restrict__ q, const T* __restrict__ k,
                                                         const T* __restrict__ v, T* __restrict__ kp, T* __restrict__ vp,
                                                         const PagedWriteParams p) {
  const int per_row = p.D / 16, heads = p.H + 2 * p.Hkv;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long rowid = id / per_row;
  if (rowid >= (long long)p.T * heads) return;
  const int c = (int)(id - rowid * per_row) * 8;
  const int t = (int)(rowid / heads), j = (int)(rowid - (long long)t * heads);
  // the token's sequence and its distance from the sequence's end
  int b, from_end;
  bool pad = false;
  if (p.cu) {
    int lo = 0, hi = p.B;       // cu[lo] <= t < cu[hi], where there is such a sequence
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.cu + mid) <= t) lo = mid; else hi = mid;
    }
    b = lo;
    from_end = __ldg(p.cu + lo + 1) - t;
    pad = from_end <= 0 || t < __ldg(p.cu + lo);
  } else {
    const int n = p.T / p.B;
    b = t / n;
    from_end = n - (t - b * n);
  }
  int pos = __ldg(p.lens + b) - from_end;
  pad = pad || pos < 0;
  T* dst;
  const T* src;
  bool rotate = true;
  if (j < p.H) {
    src = q + t * p.q_st + j * p.q_sh;
    dst = q_out + ((long long)t * p.H + j) * p.D;
  } else {
    if (pad) return;
    const int index = pos / p.page_size, page = index < p.table_width ? __ldg(p.table + b * p.table_sb + index) : -1;
    const int64_t r = pos - index * p.page_size;
    if (page < 0 || page >= p.num_pages) {
      if (p.status) atomicExch(p.status, 1);
      return;
    }
    const int hk = j - p.H;
    if (hk < p.Hkv) {
      src = k + t * p.k_st + hk * p.k_sh;
      dst = kp + page * p.kp_sp + hk * p.kp_sh + r * p.kp_sr;
    } else {
      src = v + t * p.v_st + (hk - p.Hkv) * p.v_sh;
      dst = vp + page * p.vp_sp + (hk - p.Hkv) * p.vp_sh + r * p.vp_sr;
      rotate = false;
    }
  }
  const int half = p.D / 2;
  if (pad) {
    Vec16<T> z;
#pragma unroll
    for (int e = 0; e < 8; ++e) z.v[e] = ToF<T>::from(0.f);
    st16(dst + c, z);
    st16(dst + half + c, z);
    return;
  }
  Vec16<T> lo = ld16(src + c), hi = ld16(src + half + c);
  if (rotate) {
    if (pos >= p.table_len) {
      if (p.status) atomicExch(p.status, 1);
      pos = p.table_len - 1;
    }
    const float* cs = p.cosv + (int64_t)pos * half + c;
    const float* sn = p.sinv + (int64_t)pos * half + c;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x0 = ToF<T>::to(lo.v[e]), x1 = ToF<T>::to(hi.v[e]), co = __ldg(cs + e), si = __ldg(sn + e);
      lo.v[e] = ToF<T>::from(x0 * co - x1 * si);
      hi.v[e] = ToF<T>::from(x1 * co + x0 * si);
    }
  }
  st16(dst + c, lo);
  st16(dst + half + c, hi);
}

bool rows_of_16_bytes(const void* ptr, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(ptr) & 15) return false;
  for (int64_t s : strides)
    if (s % 8 != 0) return false;
  return true;
}

template <typename T, int D, int MT>
int launch_paged(void* out, const void* q, const void* kp, const void* vp, PagedParams p, cudaStream_t stream) {
  const int rows = p.n * (p.H / p.Hkv);
  p.row_groups = (rows + 16 * MT - 1) / (16 * MT);
  const long long units = (long long)p.B * p.Hkv * p.row_groups;
  const long long cap = (long long)p.table_width * p.page_size;
  const long long keys = p.window > 0 ? std::min(cap, (long long)p.window + p.sinks + p.n) : cap;
  p.split = 1;
  static const int target = std::getenv("B200_PAGED_TARGET") ? std::atoi(std::getenv("B200_PAGED_TARGET")) : 2 * kSMs;
  while (p.split < kMaxSplit && units * p.split < target && keys > (long long)p.split * kPagedWarps * kStepKeys) p.split *= 2;
  const long long grid = units * p.split;
  if (grid > 2147483647ll) return (int)cudaErrorNotSupported;
  constexpr int smem = kPagedWarps * kWarpRing + (MT > 1 ? MT * (D / 16) * 512 : 0);
  auto kern = paged_attn_kernel<T, D, MT>;
  static OncePerDevice once;
  if (int e = once([&] {
        if (int r = opt_in_smem(kern, smem)) return r;
        return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      }))
    return e;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)p.split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kPagedWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = p.split > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (T*)out, (const T*)q, (const T*)kp, (const T*)vp, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return (int)e;
  }
  note_launch();
  return 0;
}

template <typename T>
int launch_paged(int head_dim, void* out, const void* q, const void* kp, const void* vp, const PagedParams& p, cudaStream_t stream) {
  const bool few = p.n * (p.H / p.Hkv) <= 16;
  if (head_dim == 128) return few ? launch_paged<T, 128, 1>(out, q, kp, vp, p, stream) : launch_paged<T, 128, 2>(out, q, kp, vp, p, stream);
  return few ? launch_paged<T, 64, 1>(out, q, kp, vp, p, stream) : launch_paged<T, 64, 2>(out, q, kp, vp, p, stream);
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int b200_paged_attention(const b200_paged_attn_t* a, void* out, const void* q, const void* k_pages, const void* v_pages,
                                    const int* block_table, const int* seq_lens, int* status, cudaStream_t stream) {
  if ((a->dtype != B200_BF16 && a->dtype != B200_F16) || (a->head_dim != 64 && a->head_dim != 128) || a->B <= 0 || a->n <= 0 ||
      a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv != 0 || a->page_size <= 0 || a->page_size % 16 != 0 || a->num_pages < 0 ||
      a->table_width <= 0 || (long long)a->table_width * a->page_size > 2147483647ll || a->sinks < 0)
    return (int)cudaErrorNotSupported;
  if (!rows_of_16_bytes(q, {a->q_sb, a->q_sn, a->q_sh}) || !rows_of_16_bytes(k_pages, {a->k_sp, a->k_sh, a->k_sr}) ||
      !rows_of_16_bytes(v_pages, {a->v_sp, a->v_sh, a->v_sr}) || !rows_of_16_bytes(out, {}))
    return (int)cudaErrorNotSupported;
  PagedParams p{};
  p.B = a->B; p.n = a->n; p.H = a->H; p.Hkv = a->Hkv;
  p.num_pages = a->num_pages; p.page_size = a->page_size; p.table_width = a->table_width;
  p.window = a->window; p.sinks = a->window > 0 ? a->sinks : 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.q_sb = a->q_sb; p.q_sn = a->q_sn; p.q_sh = a->q_sh;
  p.k_sp = a->k_sp; p.k_sh = a->k_sh; p.k_sr = a->k_sr;
  p.v_sp = a->v_sp; p.v_sh = a->v_sh; p.v_sr = a->v_sr;
  p.table_sb = a->table_sb;
  p.table = block_table;
  p.lens = seq_lens;
  p.status = status;
  p.page_shift = -1;
  for (int x = 4; x < 31; ++x)
    if (p.page_size == 1 << x) p.page_shift = x;
  return a->dtype == B200_BF16 ? launch_paged<__nv_bfloat16>(a->head_dim, out, q, k_pages, v_pages, p, stream)
                               : launch_paged<__half>(a->head_dim, out, q, k_pages, v_pages, p, stream);
}

extern "C" int b200_paged_rope_cache(const b200_paged_write_t* a, void* q_out, const void* q, const void* k, const void* v,
                                     const float* cosv, const float* sinv, void* k_pages, void* v_pages, const int* block_table,
                                     const int* seq_lens, const int* cu_seqlens, int* status, cudaStream_t stream) {
  if ((a->dtype != B200_BF16 && a->dtype != B200_F16) || (a->head_dim != 64 && a->head_dim != 128) || a->T <= 0 || a->B <= 0 ||
      a->H <= 0 || a->Hkv <= 0 || a->page_size <= 0 || a->num_pages < 0 || a->table_width < 0 || a->table_len <= 0 ||
      (!cu_seqlens && a->T % a->B != 0))
    return (int)cudaErrorNotSupported;
  if (!rows_of_16_bytes(q, {a->q_st, a->q_sh}) || !rows_of_16_bytes(k, {a->k_st, a->k_sh}) || !rows_of_16_bytes(v, {a->v_st, a->v_sh}) ||
      !rows_of_16_bytes(k_pages, {a->kp_sp, a->kp_sh, a->kp_sr}) || !rows_of_16_bytes(v_pages, {a->vp_sp, a->vp_sh, a->vp_sr}) ||
      !rows_of_16_bytes(q_out, {}))
    return (int)cudaErrorNotSupported;
  PagedWriteParams p{};
  p.T = a->T; p.B = a->B; p.H = a->H; p.Hkv = a->Hkv; p.D = a->head_dim;
  p.num_pages = a->num_pages; p.page_size = a->page_size; p.table_width = a->table_width; p.table_len = a->table_len;
  p.q_st = a->q_st; p.q_sh = a->q_sh; p.k_st = a->k_st; p.k_sh = a->k_sh; p.v_st = a->v_st; p.v_sh = a->v_sh;
  p.kp_sp = a->kp_sp; p.kp_sh = a->kp_sh; p.kp_sr = a->kp_sr; p.vp_sp = a->vp_sp; p.vp_sh = a->vp_sh; p.vp_sr = a->vp_sr;
  p.table_sb = a->table_sb;
  p.cosv = cosv; p.sinv = sinv;
  p.table = block_table; p.lens = seq_lens; p.cu = cu_seqlens;
  p.status = status;
  const long long threads = (long long)p.T * (p.H + 2 * p.Hkv) * (p.D / 16), grid = (threads + 255) / 256;
  if (grid > 2147483647ll) return (int)cudaErrorNotSupported;
  if (a->dtype == B200_BF16)
    paged_rope_kernel<__nv_bfloat16><<<(unsigned)grid, 256, 0, stream>>>((__nv_bfloat16*)q_out, (const __nv_bfloat16*)q,
        (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (__nv_bfloat16*)k_pages, (__nv_bfloat16*)v_pages, p);
  else
    paged_rope_kernel<__half><<<(unsigned)grid, 256, 0, stream>>>((__half*)q_out, (const __half*)q, (const __half*)k, (const __half*)v,
                                                                  (__half*)k_pages, (__half*)v_pages, p);
  B200K_LAUNCH_RET();
}
