// Attention of the newest tokens of each sequence over a paged key-value cache, and the rotary embedding that writes it.
//
// The cache is a pool of pages [num_pages, Hkv, page_size, D] for keys and one for values; row b of the block table names
// the pages of sequence b in order.  seq_lens[b] counts the tokens of the sequence that are in the cache, the newest
// included, so token i of n new ones stands at position len - n + i.  Everything that changes from step to step is read
// on the device, so that a captured step can be replayed.
// Parity: the reference has no paged cache; its decoding goes through the vendor SDPA on contiguous keys (reference
// torch_musa/csrc/aten/ops/attention/mudnn/SDP.cpp).
#include "common.cuh"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace b200k {
namespace {

// x / d for 0 <= x < 2^31 with one multiplication: m = ceil(2^(32 + s) / d) - 2^32 for s = ceil(log2 d)
struct FastDiv {
  uint32_t mul, shift;
  __device__ __forceinline__ int operator()(int x) const {
    const uint32_t h = __umulhi((uint32_t)x, mul);
    return (int)((h + (((uint32_t)x - h) >> (shift ? 1 : 0))) >> (shift ? shift - 1 : 0));
  }
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return FastDiv{(uint32_t)((((1ull << s) - d) << 32) / d + 1), s};
}

struct PagedParams {
  int B, n, H, Hkv;
  int num_pages, page_size, table_width;
  FastDiv by_page, by_heads;  // page_size; query heads of a key head
  int window, sinks;          // window <= 0: every earlier key is visible
  int split, outer;           // CTAs of a cluster and clusters that share the keys of a row group
  FastDiv by_split, by_outer;
  float* parts;               // outer > 1: [B, Hkv, rows, outer][D + 4]: a cluster's output, sum and maximum
  float scale_log2;
  int64_t q_sb, q_sn, q_sh;                    // element strides; rows of D contiguous elements
  int64_t k_sp, k_sh, k_sr, v_sp, v_sh, v_sr;  // page, head, row in the page
  int64_t table_sb;
  const int* table;
  const int* lens;
  int* status;
};

constexpr int kPagedWarps = 4;
constexpr int kPageRows = 16;          // rows of a page come in multiples of this
constexpr int kWarpRing = 16 * 1024;   // keys and values that a warp has in flight or in hand
constexpr float kRaise = 8.f;          // log2: how far a score may exceed the reference maximum

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
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
// from the shared memory of another CTA of the cluster
__device__ __forceinline__ uint32_t remote(uint32_t a, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float remote1(uint32_t a, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote(a, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 remote4(uint32_t a, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote(a, rank)) : "memory");
  return v;
}
// transposes an 8 x 8 matrix of 16-bit values that lies over the warp's registers
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void zero16(uint32_t a) { asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0) : "memory"); }
// the n lowest bits, for any n
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// d = a b + c
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
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

// The sums of an output that are NaN although no score is: an infinity met a probability that 16 bits hold as zero, or the remainder of one,
// which may be zero or negative.  What the softmax gives follows from the values that the token sees alone, its probabilities are
// positive: an infinity for those of one sign, NaN where there are both signs or a NaN.  v: four dimensions of the key head's pool.
// With finite values nobody comes here.  What its being there costs is the compiler's choice of registers: 16 sequences with 20 rows a key
// head, D 64, 15.0 us where it was 14.5; four rows or D 128 within 1 % (a second pass over the keys by the warp that
// found a NaN: 2 to 9 %).
template <typename T>
__device__ __noinline__ float4 settle_infinities(float4 sums, const T* vp, const PagedParams& p, int b, int hk, int i, int d) {
  const int pos = min(max(__ldg(p.lens + b), 0), p.table_width * p.page_size) - p.n + i;
  const int from = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int* table = p.table + b * p.table_sb;
  const T* v = vp + hk * p.v_sh + d;
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  uint32_t found[4] = {};              // 1: +inf, 2: -inf, 4: NaN
  for (int k0 = 0; k0 <= pos; k0 += kPageRows) {
    if (k0 + kPageRows <= from && k0 >= p.sinks) continue;
    const int index = p.by_page(k0), page = __ldg(table + index);
    if ((unsigned)page >= (unsigned)p.num_pages) continue;
    const T* rows = v + page * p.v_sp + (k0 - index * p.page_size) * p.v_sr;
    for (int r = 0; r < kPageRows; ++r) {
      const int j = k0 + r;
      if (j > pos || (j < from && j >= p.sinks)) continue;
      const uint2 w = *reinterpret_cast<const uint2*>(rows + r * p.v_sr);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = ((e < 2 ? w.x : w.y) >> (e & 1) * 16) & 0xffffu;
        if ((x & kExp) == kExp) found[e] |= (x & 0x7fffu) != kExp ? 4u : (x >> 15 ? 2u : 1u);
      }
    }
  }
  float o[4] = {sums.x, sums.y, sums.z, sums.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (o[e] != o[e] && (found[e] == 1u || found[e] == 2u)) o[e] = found[e] == 1u ? INFINITY : -INFINITY;
  return make_float4(o[0], o[1], o[2], o[3]);
}
// whether settle_infinities has to be asked
__device__ __forceinline__ bool unsettled(const float (&v)[4], float sum) {
  const float any = (v[0] + v[1]) + (v[2] + v[3]);        // NaN where one is (or infinities of both signs: asked in vain)
  return any != any && sum == sum;
}

// One CTA: one row group (up to 8 * NT rows = new tokens x query heads of a key head) of one (sequence, key head), one of several
// contiguous shares of the visible keys.  A share is cut into steps of 16 keys (32 when D is 64 and the rows few) that the four warps take in turn;
// each warp runs its own online softmax, the warps join through shared memory and the CTAs of a cluster through distributed shared
// memory.  A warp copies the rows of keys and of values of a step into a stage of its own ring (cp.async, whole rows at a time,
// 16-byte pieces swapped by row so that the eight rows of a matrix lie in different banks).  The products are mma m16n8k16 with the
// long side first, because a key head seldom has more than eight rows:
//   S^T = K Q^T    16 keys x 8 rows; K by ldmatrix, Q in registers;
//   O^T += V^T P^T  16 dimensions x 8 rows, 16 keys deep; V^T by ldmatrix.trans, P^T from S^T by movmatrix.
// A lane's columns are rows 2 t and 2 t + 1 in both, so a row's maximum and sum stay with the lanes that hold its outputs.  P goes in as
// a 16-bit value plus the 16-bit remainder of its rounding (2^-16 or better).  The maximum that exponents refer to is raised only
// when a score exceeds it by 2^8: then eight lanes have to be asked, which most steps leave out.
//
// What bounds it: memory, where the batch fills the machine -- 32 sequences of 1100 to 2048 keys with 32 key heads: 126 us, 830 MB read once,
// 6.6 TB/s, warps waiting for their copies (long scoreboard 5.3 of 10.9 clocks an instruction); two of 50001 to 65536 keys with 8 key heads:
// 82 us, 5.8 TB/s, on 384 of 444 places.  Where it is small, the way from the launch through length, table and keys to the joins: 3.4 us
// for 32 keys, 5.1 for 500.  With several tokens at once the same chain, longer: 16 sequences, 8 key heads, D 64, 20 rows a key head take 5.9 us
// for 8 keys (3.9 with four rows), 7.8 once two CTAs have to join (5.1), and 6.2 us more for each thousand keys (33 MB, out of the L2 cache;
// 3.3 with four rows).  Three or four warps a scheduler issue 0.34 instructions a clock; they wait for one another's results (1.8
// clocks an instruction), for copies (1.2) and at barriers (1.0).
// On the way here (us, the first two of these cases): a warp per row and scalar products 2262 / 72680; the tensor core with operands
// copied piece by piece into a lane's own slots 181 / 156 (600, then 400 instructions for 16 keys); whole rows and ldmatrix 127 / 93; keys as
// the long side of the products 124 / 82, and D 64 with four rows a key head, 64 sequences of up to 4000 keys, 62 -> 50.
// kDense: the rows of a page follow one another (the layout of the pools as they are made), so that a copy's address is a constant
// away from the page's.
template <typename T, int D, int NT, bool kDense>
__global__ void __launch_bounds__(kPagedWarps * 32, NT * D <= 256 ? 3 : 2)
paged_attn_kernel(T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ kp, const T* __restrict__ vp,
                  const __grid_constant__ PagedParams p) {
  constexpr int kRows = 8 * NT, kHalves = D == 64 && NT <= 2 ? 2 : 1, kKeys = kHalves * kPageRows, kHalf = kPageRows * D * 2;
  constexpr int kStageBytes = 2 * kHalves * kHalf, kStages = kWarpRing / kStageBytes;
  constexpr int kPad = D + 4;            // floats of a row of a part: the four lanes' rows then lie in different banks
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_m[kPagedWarps][kRows], s_l[kPagedWarps][kRows];
  __shared__ float s_top[kRows], s_sum[kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.H / p.Hkv, rows_all = p.n * G, split = p.split;
  const int cluster = p.by_split((int)blockIdx.x), rank = (int)blockIdx.x - cluster * split;      // clusters lie along x
  const int group = p.by_outer(cluster), outer = cluster - group * p.outer;
  const int r0 = group * kRows;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int rows = min(kRows, rows_all - r0);
  const int len = min(max(__ldg(p.lens + b), 0), p.table_width * p.page_size);
  // positions of the oldest and the newest token of the group; the steps that one of them sees
  const int pos0 = len - p.n + p.by_heads(r0), pos1 = len - p.n + p.by_heads(r0 + rows - 1);
  // positions of this lane's rows: 2 t and 2 t + 1 of each eight
  int pos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) pos[nt][e] = len - p.n + p.by_heads(r0 + nt * 8 + 2 * t + e);
  const int wlo = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
  const int end = pos1 >= 0 ? pos1 / kKeys + 1 : 0;
  const int sink_steps = min(end, (p.sinks + kKeys - 1) / kKeys), first = max(wlo / kKeys, sink_steps);
  const int steps = sink_steps + max(0, end - first), shares = split * p.outer, mine = outer * split + rank;
  const int s0 = (int)((long long)steps * mine / shares), s1 = (int)((long long)steps * (mine + 1) / shares);
  auto key_of = [&](int s) { return (s < sink_steps ? s : s - sink_steps + first) * kKeys; };

  const uint32_t ring = shared_u32(smem) + warp * kWarpRing;
  const int* table = p.table + b * p.table_sb;
  constexpr int kPieces = D / 8, kPerCopy = 32 / kPieces;      // 16-byte pieces of a row, rows that one instruction copies
  const int crow = lane / kPieces, cpiece = lane % kPieces;
  const T* kbase = kp + hk * p.k_sh + crow * p.k_sr + cpiece * 8;
  const T* vbase = vp + hk * p.v_sh + crow * p.v_sr + cpiece * 8;
  constexpr int kSwaps = 8 / kPerCopy;   // rows r of copy i: their swap depends on i modulo this
  uint32_t cdst[kSwaps];
#pragma unroll
  for (int i = 0; i < kSwaps; ++i) cdst[i] = (uint32_t)(crow * D * 2 + ((cpiece ^ ((i * kPerCopy + crow) & 7)) * 16));
  const int mi = lane >> 3, mr = lane & 7;
  // a lane's row address in a stage for ldmatrix; the piece 2 x of a row is at ((2 x) ^ swap) * 16, for x < 4
  uint32_t kaddr[4], vaddr[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    kaddr[x] = ring + (uint32_t)(((mi & 1) * 8 + mr) * D * 2) + (((uint32_t)x * 32) ^ (uint32_t)(((mi >> 1) ^ mr) * 16));
    vaddr[x] = ring + (uint32_t)(kHalves * kHalf + ((mi >> 1) * 8 + mr) * D * 2) + (((uint32_t)x * 32) ^ (uint32_t)(((mi & 1) ^ mr) * 16));
  }

  // A step's page numbers, read one step before they are needed; kNoPage for a half in which nobody sees a key: the table's entry may then
  // be anything.
  constexpr int kNoPage = -0x7fffffff - 1;
  struct Pages { int n[kHalves]; };
  auto entry = [&](int s) {
    Pages e;
    const int k0 = key_of(s);
#pragma unroll
    for (int x = 0; x < kHalves; ++x) {
      const int kx = k0 + x * kPageRows;
      const bool seen = s < s1 && kx <= pos1 && (kHalves == 1 || kx + kPageRows > wlo || kx < p.sinks);
      e.n[x] = seen ? max(__ldg(table + p.by_page(kx)), -1) : kNoPage;
    }
    return e;
  };
  uint32_t found = 0;                // one bit a stage and half: whether its page is in the pool
  auto issue = [&](int s, const Pages& e, int stage) {
    if (s < s1) {
#pragma unroll
      for (int x = 0; x < kHalves; ++x) {
        const int k0 = key_of(s) + x * kPageRows, number = e.n[x];
        const bool there = (unsigned)number < (unsigned)p.num_pages;
        if (!there && number != kNoPage && lane == 0 && p.status) atomicExch(p.status, 1);
        const uint32_t bit = 1u << (stage * kHalves + x);
        found = there ? found | bit : found & ~bit;
        const uint32_t page = there ? (uint32_t)number : 0u, row = (uint32_t)(k0 - p.by_page(k0) * p.page_size);
        const T* ks = kbase + (uint64_t)page * (uint64_t)p.k_sp + (kDense ? row * D : (uint64_t)row * (uint64_t)p.k_sr);
        const T* vs = vbase + (uint64_t)page * (uint64_t)p.v_sp + (kDense ? row * D : (uint64_t)row * (uint64_t)p.v_sr);
        const uint32_t dst = ring + stage * kStageBytes + x * kHalf;
        const int n16 = there ? 16 : 0;        // a page that is not there: zeros
#pragma unroll
        for (int i = 0; i < kPageRows / kPerCopy; ++i) {
          const uint32_t d = dst + cdst[i % kSwaps] + (uint32_t)(i * kPerCopy * D * 2);
          copy16(d, ks + (kDense ? i * kPerCopy * D : i * kPerCopy * p.k_sr), n16);
          copy16(d + kHalves * kHalf, vs + (kDense ? i * kPerCopy * D : i * kPerCopy * p.v_sr), n16);
        }
      }
    }
    copy_commit();
  };
  // Q as operands: row g of each eight, dimensions 16 ks + 2 t and 8 further
  uint32_t qf[NT][D / 16][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g, i = p.by_heads(r0 + r);
    const T* row = q + b * p.q_sb + i * p.q_sn + (hk * G + r0 + r - i * G) * p.q_sh + 2 * t;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[nt][ks][e] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(row + ks * 16 + e * 8)) : 0u;
  }

  float o[NT][D / 16][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int x = 0; x < D / 16; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][x][e] = 0.f;
    m_run[nt][0] = m_run[nt][1] = -INFINITY;
    l_run[nt][0] = l_run[nt][1] = 0.f;
  }

  // The first passes only fill the ring, so that the code of the copies is there once: a CTA has few steps, and code that it meets
  // for the first time costs more than what it does.
  Pages number = entry(s0 + warp);
  int stage = 0;
  for (int s = s0 + warp - kStages * kPagedWarps; s < s1; s += kPagedWarps) {
    if (s >= s0) {
    copy_wait<kStages - 1>();
    __syncwarp();
    const int k0 = key_of(s);
    const uint32_t at = stage * kStageBytes;
    const uint32_t ka[4] = {kaddr[0] + at, kaddr[1] + at, kaddr[2] + at, kaddr[3] + at};
    const uint32_t va[4] = {vaddr[0] + at, vaddr[1] + at, vaddr[2] + at, vaddr[3] + at};
    float sc[kHalves][NT][4];            // key g (and g + 8) of a half, rows 2 t and 2 t + 1
    {
      constexpr int kChains = kHalves * NT >= 4 ? 1 : 4 / (kHalves * NT);      // independent sums in flight: four at least
      float part[kChains][kHalves][NT][4];
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int x = 0; x < kHalves; ++x) {
          const uint4 kf = ldmatrix(ka[ks & 3] + (ks >> 2) * 128 + x * kHalf);
          const uint32_t a[4] = {kf.x, kf.y, kf.z, kf.w};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float(&d)[4] = part[ks % kChains][x][nt];
            if (ks < kChains) mma16816<T>(d, a, qf[nt][ks][0], qf[nt][ks][1], zero);
            else mma16816<T>(d, a, qf[nt][ks][0], qf[nt][ks][1], d);
          }
        }
#pragma unroll
      for (int x = 0; x < kHalves; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[x][nt][e] = part[0][x][nt][e];
#pragma unroll
            for (int c = 1; c < kChains; ++c) sc[x][nt][e] += part[c][x][nt][e];
          }
    }
    // V^T of dimensions [16 j, 16 j + 16) and the keys of half x
    auto values = [&](int j, int x) { return ldmatrix_t(va[j & 3] + (j >> 2) * 128 + x * kHalf); };
    const uint32_t pages = (found >> (stage * kHalves)) & ((1u << kHalves) - 1u);
    const bool all = pages == (1u << kHalves) - 1u && k0 + kKeys - 1 <= pos0 && (p.window <= 0 || k0 > pos1 - p.window || k0 + kKeys <= p.sinks);
    // bit j: a token at position ps sees key k0 + j
    auto sees = [&](int ps) {
      const uint32_t there = kHalves == 1 ? (pages ? 0xffffu : 0u) : (pages & 1u ? 0xffffu : 0u) | (pages & 2u ? 0xffff0000u : 0u);
      return there & low_bits(ps + 1 - k0) & ~(p.window > 0 ? low_bits(ps - p.window + 1 - k0) & ~low_bits(p.sinks - k0) : 0u);
    };
    bool careful = false;
    if (!all) {
      // Values that no row sees become zero: with a probability of zero nothing else would be safe.
      // Some row sees a key when it is not past the newest token, and a sink or not in front of the oldest one's window.
      const uint32_t unseen = ~(low_bits(pos1 + 1 - k0) & ~(low_bits(wlo - k0) & ~low_bits(p.sinks - k0))) & (kKeys == 32 ? ~0u : 0xffffu);
      if (unseen) {
#pragma unroll
        for (int i = 0; i < kKeys / kPerCopy; ++i)
          if ((unseen >> (i * kPerCopy + crow)) & 1u)
            zero16(ring + at + kHalves * kHalf + (uint32_t)(crow * D * 2 + cpiece * 16 + i * kPerCopy * D * 2));
        __syncwarp();
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = sees(pos[nt][e]) >> g;
#pragma unroll
          for (int x = 0; x < kHalves; ++x)
#pragma unroll
            for (int k8 = 0; k8 < 2; ++k8)
              if (!((w >> (x * 16 + k8 * 8)) & 1u)) sc[x][nt][k8 * 2 + e] = -INFINITY;
        }
      if (pos0 != pos1) {            // rows differ in what they see
        bool odd = false;
#pragma unroll 1
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int x = 0; x < kHalves; ++x) {
            const uint4 v = ldmatrix_t((j & 2 ? (j & 1 ? va[3] : va[2]) : (j & 1 ? va[1] : va[0])) + (j >> 2) * 128 + x * kHalf);
            odd = odd || not_finite<T>(v.x) || not_finite<T>(v.y) || not_finite<T>(v.z) || not_finite<T>(v.w);
          }
        careful = __any_sync(0xffffffffu, odd);
      }
    }
    // a score that exceeds the reference by 2^8: every row's maximum is found and becomes the reference
    bool above = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(sc[0][nt][e], sc[0][nt][e + 2]);
        if constexpr (kHalves == 2) x = fmaxf(x, fmaxf(sc[1][nt][e], sc[1][nt][e + 2]));
        above = above || x * p.scale_log2 > m_run[nt][e] + kRaise;
      }
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(sc[0][nt][e], sc[0][nt][e + 2]);
          if constexpr (kHalves == 2) x = fmaxf(x, fmaxf(sc[1][nt][e], sc[1][nt][e + 2]));
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
          const float m_new = fmaxf(m_run[nt][e], x * p.scale_log2);
          const float alpha = m_new == -INFINITY ? 1.f : exp2_fast(m_run[nt][e] - m_new);
          m_run[nt][e] = m_new;
          l_run[nt][e] *= alpha;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            o[nt][j][e] *= alpha;
            o[nt][j][e + 2] *= alpha;
          }
        }
    }
    uint32_t hi[kHalves][NT][2], lo[kHalves][NT][2];      // P^T: keys 2 t.. and 2 t + 8.. of row g
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float ref0 = m_run[nt][0] == -INFINITY ? 0.f : m_run[nt][0], ref1 = m_run[nt][1] == -INFINITY ? 0.f : m_run[nt][1];
#pragma unroll
      for (int x = 0; x < kHalves; ++x)
#pragma unroll
        for (int k8 = 0; k8 < 2; ++k8) {
          const float p0 = exp2_fast(fmaf(sc[x][nt][k8 * 2], p.scale_log2, -ref0)), p1 = exp2_fast(fmaf(sc[x][nt][k8 * 2 + 1], p.scale_log2, -ref1));
          l_run[nt][0] += p0;
          l_run[nt][1] += p1;
          uint32_t h, l;
          split2<T>(p0, p1, h, l);
          hi[x][nt][k8] = transpose8(h);
          lo[x][nt][k8] = transpose8(l);
        }
    }
    if (!careful) {
      constexpr int kBatch = 4;            // operands in hand: the two products of an output are four or more apart
#pragma unroll
      for (int j0 = 0; j0 < D / 16; j0 += kBatch)
#pragma unroll
        for (int x = 0; x < kHalves; ++x) {
          uint4 v[kBatch];
#pragma unroll
          for (int j = 0; j < kBatch; ++j) v[j] = values(j0 + j, x);
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
              const uint32_t a[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint32_t(&w)[2] = part ? lo[x][nt] : hi[x][nt];
                mma16816<T>(o[nt][j0 + j], a, w[0], w[1], o[nt][j0 + j]);
              }
            }
        }
    } else {
      // An infinity or a NaN among values that some rows see and others do not: token by token, with the values that the token
      // does not see as zeros, and only its own rows kept.
#pragma unroll 1
      for (int ps = pos0; ps <= pos1; ++ps) {
#pragma unroll
        for (int x = 0; x < kHalves; ++x) {
          const uint32_t w = sees(ps) >> (x * 16 + 2 * t);
          const uint32_t see0 = (w & 1u ? 0xffffu : 0u) | (w & 2u ? 0xffff0000u : 0u);
          const uint32_t see1 = (w & 0x100u ? 0xffffu : 0u) | (w & 0x200u ? 0xffff0000u : 0u);
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            const uint4 v = values(j, x);
            const uint32_t a[4] = {v.x & see0, v.y & see0, v.z & see1, v.w & see1};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float zero[4] = {0.f, 0.f, 0.f, 0.f};
              float acc[4];
              mma16816<T>(acc, a, hi[x][nt][0], hi[x][nt][1], zero);
              mma16816<T>(acc, a, lo[x][nt][0], lo[x][nt][1], acc);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (pos[nt][e & 1] == ps) o[nt][j][e] += acc[e];
            }
          }
        }
      }
    }
    __syncwarp();
    }
    const Pages now = number;
    number = entry(s + (kStages + 1) * kPagedWarps);
    issue(s + kStages * kPagedWarps, now, stage);
    if (++stage == kStages) stage = 0;
  }

  // ---- the warps' parts: maxima and sums first, then the outputs relative to the common maximum
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[nt][e];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
      if (g == 0) {
        s_m[warp][nt * 8 + 2 * t + e] = m_run[nt][e];
        s_l[warp][nt * 8 + 2 * t + e] = l;
      }
    }
  copy_wait<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);            // [warps][kRows][kPad]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * t + e;
      if (r >= rows) continue;
      float top = s_m[0][r];
#pragma unroll
      for (int w = 1; w < kPagedWarps; ++w) top = fmaxf(top, s_m[w][r]);
      const float f = m_run[nt][e] == -INFINITY ? 1.f : exp2_fast(m_run[nt][e] - top);   // no key: zeros, or NaN
      if (warp == 0 && g == 0) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kPagedWarps; ++w) sum += s_m[w][r] == -INFINITY ? s_l[w][r] : s_l[w][r] * exp2_fast(s_m[w][r] - top);
        s_top[r] = top;
        s_sum[r] = sum;
      }
      float* dst = part + ((size_t)warp * kRows + r) * kPad + g;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        dst[j * 16] = o[nt][j][e] * f;
        dst[j * 16 + 8] = o[nt][j][e + 2] * f;
      }
    }
  __syncthreads();
  auto store = [&](int r, int d, float (&v)[4], float sum, float top) {
    if (p.outer > 1) {
      float* dst = p.parts + ((((int64_t)b * p.Hkv + hk) * rows_all + r0 + r) * p.outer + outer) * (D + 4);
      *reinterpret_cast<float4*>(dst + d) = make_float4(v[0], v[1], v[2], v[3]);
      if (d == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(sum, top);
      return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;       // no key: zeros
    const int i = p.by_heads(r0 + r), h = hk * G + r0 + r - i * G;
    if (unsettled(v, sum)) {
      const float4 x = settle_infinities<T>(make_float4(v[0], v[1], v[2], v[3]), vp, p, b, hk, i, d);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
    T o4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o4[e] = ToF<T>::from(sum == 0.f ? 0.f : v[e] * inv);
    *reinterpret_cast<uint2*>(out + (((int64_t)b * p.n + i) * p.H + h) * D + d) = *reinterpret_cast<const uint2*>(o4);
  };
  for (int x = threadIdx.x; x < rows * (D / 4); x += kPagedWarps * 32) {       // the CTA's sum, over warp 0's part
    const int r = x / (D / 4), d = x % (D / 4) * 4;
    float4 v = *reinterpret_cast<const float4*>(part + r * kPad + d);
#pragma unroll
    for (int w = 1; w < kPagedWarps; ++w) {
      const float4 y = *reinterpret_cast<const float4*>(part + (w * kRows + r) * kPad + d);
      v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
    }
    if (split == 1) {
      float v4[4] = {v.x, v.y, v.z, v.w};
      store(r, d, v4, s_sum[r], s_top[r]);
    } else {
      *reinterpret_cast<float4*>(part + r * kPad + d) = v;
    }
  }
  if (split == 1) return;
  // ---- the cluster's parts: every CTA finishes its share of the elements
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const uint32_t a_top = shared_u32(s_top), a_sum = shared_u32(s_sum), a_part = shared_u32(part);
  const int quads = rows * D / 4, share = (quads + split - 1) / split;
  for (int x = rank * share + threadIdx.x; x < min(quads, (rank + 1) * share); x += kPagedWarps * 32) {
    const int r = x / (D / 4), d = x % (D / 4) * 4;
    float top = -INFINITY, sum = 0.f, v[4] = {};
    // four CTAs at a time, all their loads in flight; relative to the maximum so far, as always
    for (int c0 = 0; c0 < split; c0 += 4) {
      float mc[4], lc[4];
      float4 y[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mc[c] = -INFINITY;
        lc[c] = 0.f;
        y[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c0 + c < split) {
          mc[c] = remote1(a_top + r * 4, c0 + c);
          lc[c] = remote1(a_sum + r * 4, c0 + c);
          y[c] = remote4(a_part + (r * kPad + d) * 4, c0 + c);
        }
      }
      const float up = fmaxf(fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])), top);
      const float old = top == -INFINITY ? 1.f : exp2_fast(top - up);
      top = up;
      sum *= old;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= old;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float f = mc[c] == -INFINITY ? 1.f : exp2_fast(mc[c] - up);      // a CTA without a key has zeros
        sum += lc[c] * f;
        v[0] += y[c].x * f; v[1] += y[c].y * f; v[2] += y[c].z * f; v[3] += y[c].w * f;
      }
    }
    store(r, d, v, sum, top);
  }
  // nobody leaves while its memory may still be read
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Joins the clusters' parts of a row: a thread owns four dimensions of one row.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_join_kernel(T* __restrict__ out, const T* __restrict__ vp,
                                                         const __grid_constant__ PagedParams p) {
  const int G = p.H / p.Hkv, rows_all = p.n * G;
  const int64_t x = (int64_t)blockIdx.x * 128 + threadIdx.x, row = x / (D / 4);
  if (row >= (int64_t)p.B * p.Hkv * rows_all) return;
  const int d = (int)(x % (D / 4)) * 4;
  const float* src = p.parts + row * p.outer * (D + 4);
  float top = -INFINITY, sum = 0.f, v[4] = {};
  for (int c = 0; c < p.outer; ++c) top = fmaxf(top, src[c * (D + 4) + D + 1]);
  for (int c = 0; c < p.outer; ++c) {
    const float4 y = *reinterpret_cast<const float4*>(src + c * (D + 4) + d);
    const float2 st = *reinterpret_cast<const float2*>(src + c * (D + 4) + D);
    const float f = st.y == -INFINITY ? 1.f : exp2_fast(st.y - top);
    sum += st.x * f;
    v[0] += y.x * f; v[1] += y.y * f; v[2] += y.z * f; v[3] += y.w * f;
  }
  const int64_t unit = row / rows_all;
  const int r = (int)(row - unit * rows_all), i = p.by_heads(r), hk = (int)(unit % p.Hkv), h = hk * G + r - i * G;
  if (unsettled(v, sum)) {
    const float4 x = settle_infinities<T>(make_float4(v[0], v[1], v[2], v[3]), vp, p, (int)(unit / p.Hkv), hk, i, d);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  }
  T o4[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) o4[e] = ToF<T>::from(sum == 0.f ? 0.f : v[e] / sum);
  *reinterpret_cast<uint2*>(out + ((unit / p.Hkv * p.n + i) * p.H + h) * D + d) = *reinterpret_cast<const uint2*>(o4);
}

struct PagedWriteParams {
  int T, B, H, Hkv;
  int rows, per_sequence;     // T * (H + 2 * Hkv); T / B
  FastDiv by_row, by_token, by_page;
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

// q_out = rotate(q); rotate(k) and v go to their rows of the cache.  A thread owns eight adjacent dimensions of the first half of one
// row and their partners in the second half.  Its two loads are on their way before the position and the page are looked up, one
// load after the other.  Bound by memory: 14.8 us for 4096 prompt tokens with 32 + 2 x 8 heads replayed from a graph (101 MB, 6.8 TB/s, a
// part of it in the L2 cache), 20.4 with other inputs each time.  A block per token, whose threads share the look-up and go over
// several heads, was slower (19.4 in a graph: fewer loads in flight), and so were 64-bit divisions in place of the multiplications (17.6).
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_rope_kernel(T* __restrict__ q_out, const T* __restrict__ q, const T* __restrict__ k,
                                                         const T* __restrict__ v, T* __restrict__ kp, T* __restrict__ vp,
                                                         const PagedWriteParams p) {
  constexpr int kPerRow = D / 16, half = D / 2;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (int64_t)p.rows * kPerRow) return;
  const int row = (int)(id / kPerRow), c = (int)(id % kPerRow) * 8;
  const int t = p.by_row(row), j = row - t * (p.H + 2 * p.Hkv), jk = j - p.H, jv = jk - p.Hkv;
  const T* src = (j < p.H ? q + t * p.q_st + j * p.q_sh : jv < 0 ? k + t * p.k_st + jk * p.k_sh : v + t * p.v_st + jv * p.v_sh) + c;
  Vec16<T> lo = ld16_stream(src), hi = ld16_stream(src + half);
  // the token's sequence and its distance from the sequence's end
  int b, from_end;
  bool pad = false;
  if (p.cu) {
    int lo_b = 0, hi_b = p.B;       // cu[lo_b] <= t < cu[hi_b], where there is such a sequence
    while (hi_b - lo_b > 1) {
      const int mid = (lo_b + hi_b) >> 1;
      if (__ldg(p.cu + mid) <= t) lo_b = mid; else hi_b = mid;
    }
    b = lo_b;
    from_end = __ldg(p.cu + b + 1) - t;
    pad = from_end <= 0 || t < __ldg(p.cu + b);
  } else {
    b = p.by_token(t);
    from_end = (b + 1) * p.per_sequence - t;
  }
  int pos = __ldg(p.lens + b) - from_end;
  pad = pad || pos < 0;
  T* dst = q_out + ((int64_t)t * p.H + j) * D + c;
  if (j >= p.H) {
    if (pad) return;
    const int index = p.by_page(pos), page = index < p.table_width ? __ldg(p.table + b * p.table_sb + index) : -1;
    if ((unsigned)page >= (unsigned)p.num_pages) {
      if (p.status) atomicExch(p.status, 1);
      return;
    }
    const int64_t r = pos - index * p.page_size;
    dst = (jv < 0 ? kp + page * p.kp_sp + jk * p.kp_sh + r * p.kp_sr : vp + page * p.vp_sp + jv * p.vp_sh + r * p.vp_sr) + c;
  }
  if (jv < 0) {
    if (pos >= p.table_len && p.status) atomicExch(p.status, 1);
    const int64_t at = (int64_t)min(max(pos, 0), p.table_len - 1) * half + c;
#pragma unroll
    for (int e4 = 0; e4 < 8; e4 += 4) {
      const float4 co4 = __ldg(reinterpret_cast<const float4*>(p.cosv + at + e4)), si4 = __ldg(reinterpret_cast<const float4*>(p.sinv + at + e4));
      const float co[4] = {co4.x, co4.y, co4.z, co4.w}, si[4] = {si4.x, si4.y, si4.z, si4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = ToF<T>::to(lo.v[e4 + e]), x1 = ToF<T>::to(hi.v[e4 + e]);
        lo.v[e4 + e] = ToF<T>::from(pad ? 0.f : x0 * co[e] - x1 * si[e]);
        hi.v[e4 + e] = ToF<T>::from(pad ? 0.f : x1 * co[e] + x0 * si[e]);
      }
    }
  }
  st16(dst, lo);
  st16(dst + half, hi);
}

bool rows_of_16_bytes(const void* ptr, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(ptr) & 15) return false;
  for (int64_t s : strides)
    if (s % 8 != 0) return false;
  return true;
}

// How the keys of a row group are shared: CTAs of a cluster, and clusters whose parts a second kernel joins.
struct PagedPlan {
  int tiles;          // eights of rows of a CTA
  long long groups;   // row groups of a (sequence, key head)
  int split, outer;
};
PagedPlan paged_plan(const b200_paged_attn_t* a) {
  PagedPlan p{};
  const long long eights = ((long long)a->n * (a->H / a->Hkv) + 7) / 8;
  p.groups = (eights + 3) / 4;
  p.tiles = (int)((eights + p.groups - 1) / p.groups);
  const long long units = (long long)a->B * a->Hkv * p.groups, cap = (long long)a->table_width * a->page_size;
  const long long keys = a->window > 0 ? std::min(cap, (long long)a->window + a->sinks + a->n) : cap;
  const long long slots = kSMs * (p.tiles * a->head_dim <= 256 ? 3 : 2);      // CTAs that are resident at once
  const long long most = std::max(1ll, keys / 64);            // a step for every warp of a share
  p.outer = 1;
  // Few rows over a long length: sixteen CTAs a unit would leave SMs idle.  (One sequence of 65536 keys with one key head: 64 us with one
  // cluster, 18 with 32 of eight; but 4000 keys with eight key heads 9 us with clusters of 16, 12 with three a unit, for the second kernel.)
  if (units * 16 < 2 * kSMs && keys > 16 * 1024) {
    const long long shares = std::max(1ll, std::min(slots / units, keys / 256));
    p.outer = (int)((shares + 7) / 8);
    p.split = (int)(shares / p.outer);
  } else {
    // clusters of more than eight leave about a quarter of the places empty (a cluster lies within one group of SMs)
    const long long one_wave = std::max(std::min(slots / units, 8ll), slots * 3 / 4 / units);
    // one wave where it fits, else two CTAs a unit while that is less than four waves: shorter pieces even out different lengths (512 units of
    // 100 to 4000 keys: 95 us whole, 88 halved, 98 in fours; 256 units with 20 rows: 86 / 77 / 80)
    p.split = (int)std::min({std::max(one_wave, units < 2 * slots ? 2ll : 1ll), most, 16ll});
  }
  return p;
}

template <typename T, int D, int NT, bool kDense>
int launch_paged(const PagedPlan& plan, void* out, const void* q, const void* kp, const void* vp, const PagedParams& p, cudaStream_t stream) {
  constexpr int smem = kPagedWarps * std::max<int>(kWarpRing, 8 * NT * (D + 4) * 4);
  auto kern = paged_attn_kernel<T, D, NT, kDense>;
  static OncePerDevice once;
  if (int e = once([&] {
        if (int r = opt_in_smem(kern, smem)) return r;
        return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      }))
    return e;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)plan.split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(plan.groups * plan.split * plan.outer), (unsigned)p.Hkv, (unsigned)p.B);
  cfg.blockDim = dim3(kPagedWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = plan.split > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (T*)out, (const T*)q, (const T*)kp, (const T*)vp, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return (int)e;
  }
  note_launch();
  if (plan.outer == 1) return 0;
  const long long threads = (long long)p.B * p.Hkv * p.n * (p.H / p.Hkv) * (D / 4);
  paged_join_kernel<T, D><<<(unsigned)((threads + 127) / 128), 128, 0, stream>>>((T*)out, (const T*)vp, p);
  B200K_LAUNCH_RET();
}

template <typename T, int D>
int launch_paged(const PagedPlan& plan, void* out, const void* q, const void* kp, const void* vp, const PagedParams& p, cudaStream_t stream) {
  const bool dense = p.k_sr == D && p.v_sr == D;
#define B200_PAGED_LAUNCH(NT) \
  return dense ? launch_paged<T, D, NT, true>(plan, out, q, kp, vp, p, stream) : launch_paged<T, D, NT, false>(plan, out, q, kp, vp, p, stream)
  switch (plan.tiles) {
    case 1: B200_PAGED_LAUNCH(1);
    case 2: B200_PAGED_LAUNCH(2);
    case 3: B200_PAGED_LAUNCH(3);
    default: B200_PAGED_LAUNCH(4);
  }
#undef B200_PAGED_LAUNCH
}

bool paged_sizes_ok(const b200_paged_attn_t* a) {
  return (a->dtype == B200_BF16 || a->dtype == B200_F16) && (a->head_dim == 64 || a->head_dim == 128) && a->B > 0 && a->n > 0 && a->H > 0 &&
         a->Hkv > 0 && a->H % a->Hkv == 0 && a->page_size > 0 && a->page_size % kPageRows == 0 && a->num_pages >= 0 && a->table_width > 0 &&
         (long long)a->table_width * a->page_size <= (1 << 30) && a->n <= (1 << 29) && a->sinks >= 0 && a->B <= 65535 && a->Hkv <= 65535 &&
         (long long)a->n * (a->H / a->Hkv) <= (1 << 24);
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int64_t b200_paged_attention_workspace(const b200_paged_attn_t* a) {
  if (!paged_sizes_ok(a)) return 0;
  const PagedPlan plan = paged_plan(a);
  return plan.outer > 1 ? (int64_t)a->B * a->H * a->n * plan.outer * (a->head_dim + 4) : 0;
}

extern "C" int b200_paged_attention(const b200_paged_attn_t* a, void* out, const void* q, const void* k_pages, const void* v_pages,
                                    const int* block_table, const int* seq_lens, float* workspace, int* status, cudaStream_t stream) {
  if (!paged_sizes_ok(a)) return (int)cudaErrorNotSupported;
  if (!rows_of_16_bytes(q, {a->q_sb, a->q_sn, a->q_sh}) || !rows_of_16_bytes(k_pages, {a->k_sp, a->k_sh, a->k_sr}) ||
      !rows_of_16_bytes(v_pages, {a->v_sp, a->v_sh, a->v_sr}) || !rows_of_16_bytes(out, {}))
    return (int)cudaErrorNotSupported;
  PagedParams p{};
  p.B = a->B; p.n = a->n; p.H = a->H; p.Hkv = a->Hkv;
  p.num_pages = a->num_pages; p.page_size = a->page_size; p.table_width = a->table_width;
  p.window = std::min(a->window, 1 << 30);             // differences of positions stay in 32 bits
  p.sinks = a->window > 0 ? std::min(a->sinks, 1 << 30) : 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.q_sb = a->q_sb; p.q_sn = a->q_sn; p.q_sh = a->q_sh;
  p.k_sp = a->k_sp; p.k_sh = a->k_sh; p.k_sr = a->k_sr;
  p.v_sp = a->v_sp; p.v_sh = a->v_sh; p.v_sr = a->v_sr;
  p.table_sb = a->table_sb;
  p.table = block_table;
  p.lens = seq_lens;
  p.status = status;
  const PagedPlan plan = paged_plan(a);
  if (plan.outer > 1 && !workspace) return (int)cudaErrorInvalidValue;
  if (plan.groups * plan.split * plan.outer > 2147483647ll) return (int)cudaErrorNotSupported;
  p.by_page = fast_div((uint32_t)p.page_size);
  p.by_heads = fast_div((uint32_t)(p.H / p.Hkv));
  p.split = plan.split;
  p.outer = plan.outer;
  p.by_split = fast_div((uint32_t)plan.split);
  p.by_outer = fast_div((uint32_t)plan.outer);
  p.parts = workspace;
  const bool wide = a->head_dim == 128;
  if (a->dtype == B200_BF16)
    return wide ? launch_paged<__nv_bfloat16, 128>(plan, out, q, k_pages, v_pages, p, stream)
                : launch_paged<__nv_bfloat16, 64>(plan, out, q, k_pages, v_pages, p, stream);
  return wide ? launch_paged<__half, 128>(plan, out, q, k_pages, v_pages, p, stream)
              : launch_paged<__half, 64>(plan, out, q, k_pages, v_pages, p, stream);
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
      !rows_of_16_bytes(q_out, {}) || !rows_of_16_bytes(cosv, {}) || !rows_of_16_bytes(sinv, {}))
    return (int)cudaErrorNotSupported;
  PagedWriteParams p{};
  p.T = a->T; p.B = a->B; p.H = a->H; p.Hkv = a->Hkv;
  p.num_pages = a->num_pages; p.page_size = a->page_size; p.table_width = a->table_width; p.table_len = a->table_len;
  p.q_st = a->q_st; p.q_sh = a->q_sh; p.k_st = a->k_st; p.k_sh = a->k_sh; p.v_st = a->v_st; p.v_sh = a->v_sh;
  p.kp_sp = a->kp_sp; p.kp_sh = a->kp_sh; p.kp_sr = a->kp_sr; p.vp_sp = a->vp_sp; p.vp_sh = a->vp_sh; p.vp_sr = a->vp_sr;
  p.table_sb = a->table_sb;
  p.cosv = cosv; p.sinv = sinv;
  p.table = block_table; p.lens = seq_lens; p.cu = cu_seqlens;
  p.status = status;
  const long long rows = (long long)p.T * (p.H + 2ll * p.Hkv), grid = (rows * (a->head_dim / 16) + 255) / 256;
  if (rows > 2147483647ll || grid > 2147483647ll) return (int)cudaErrorNotSupported;
  p.rows = (int)rows;
  p.per_sequence = p.T / p.B;
  p.by_row = fast_div((uint32_t)(p.H + 2 * p.Hkv));
  p.by_token = fast_div((uint32_t)std::max(1, p.per_sequence));
  p.by_page = fast_div((uint32_t)p.page_size);
  auto launch = [&](auto kern, auto* qo) {
    using T = std::remove_pointer_t<decltype(qo)>;
    kern<<<(unsigned)grid, 256, 0, stream>>>(qo, (const T*)q, (const T*)k, (const T*)v, (T*)k_pages, (T*)v_pages, p);
  };
  const bool wide = a->head_dim == 128;
  if (a->dtype == B200_BF16)
    wide ? launch(paged_rope_kernel<__nv_bfloat16, 128>, (__nv_bfloat16*)q_out) : launch(paged_rope_kernel<__nv_bfloat16, 64>, (__nv_bfloat16*)q_out);
  else
    wide ? launch(paged_rope_kernel<__half, 128>, (__half*)q_out) : launch(paged_rope_kernel<__half, 64>, (__half*)q_out);
  B200K_LAUNCH_RET();
}
