// Flash-attention forward on the 5th-generation tensor cores (head_dim 128, bf16 / fp16, optional causal mask or sliding
// window with sinks, grouped-query heads): two query tiles per CTA in ping-pong, scores and the output accumulators in TMEM, K / V through
// a TMA ring, every mbarrier wait bounded (status word as for the GEMMs).  The kernel comment below has the pipeline.
//
// Parity: the reference calls a closed vendor flash kernel (reference torch_musa/csrc/aten/ops/attention/mudnn/SDP.cpp:470-673).
#include "attention_common.cuh"

#include <algorithm>
#include <type_traits>

namespace b200k {
namespace {
using namespace gemmdev;
using namespace attndev;

constexpr int AQ = 128, AK = 128, AD = 128;          // query rows per tile, keys per block, head dim
constexpr int kTile = 128 * 128 * 2;                  // 32 KB: any of Q, K, V
constexpr int kRing = 5;                              // K / V tiles in flight
constexpr int kAttnSmem = 2 * kTile /*Q0,Q1*/ + kRing * kTile + 1024 + 512 /*barriers, units*/;
constexpr int kAttnThreads = 384;                     // 2 softmax warpgroups; one with the TMA, the MMA and the unit warp
constexpr int kUnitReaders = 10;                      // kWin: the TMA, MMA and softmax warps, which the unit warp tells what to do
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;    // after the split: a row of scores stays in registers
constexpr int kLaunchRegs = (2 * kSoftmaxRegs + kOtherRegs + 2) / 3;   // what the launch has to bring for that split
constexpr uint32_t kAttnTmemCols = 512;               // S0, S1, O0, O1
constexpr int kFirstPart = 64;                        // keys of a block whose P is released before the rest is computed
constexpr float kRescaleThreshold = 8.f;              // log2 domain: P stays below 2^8

struct AttnParams {
  int B, H, Hkv, Sq, Sk;
  int causal;
  float scale_log2;           // softmax scale * log2(e)
  int64_t o_sb, o_sh, o_ss;   // output strides in elements (last dim contiguous)
  float* lse;                 // [B, H, Sq]; packed sequences: [H, total_q]
  int q_blocks, q_pairs;
  // packed variable-length sequences (NULL: dense batch): sequence b holds rows [cu_q[b], cu_q[b + 1]) of the packed
  // q / out [total_q, H, 128] and rows [cu_k[b], cu_k[b + 1]) of k / v; Sq / Sk are then the longest lengths
  const int* cu_q;
  const int* cu_k;
  int total_q;
  int* status;
  int units;                  // pairs of query tiles of all (batch, head) instances
  void* remainder;            // kWin: what rounding left of the output, laid out like it, or NULL
  int window, sinks;          // kWin: key j is visible when j <= i and (i - j < window or j < sinks)
};

// One CTA owns two adjacent 128-row query tiles of one (batch, head).  Per block of 128 keys and per tile t:
//   S_t = Q_t K^T     tcgen05.mma M128 N128 K16 x 8 into TMEM (operands in 128B-swizzled shared memory);
//   softmax           warpgroup t, one query row per thread: the row of S comes into registers once, P = exp2(S * scale - m)
//                     goes back as 16-bit pairs into TMEM over the columns of S, the block maximum is found on the side;
//   O_t += P_t V      tcgen05.mma with A = P from TMEM, accumulating in TMEM over all key blocks.
// P never touches shared memory: the M128 N128 products with both operands there already take all of its 128 bytes per
// clock, and writing P there, fencing the async proxy and reading it back stood in the middle of the chain S -> softmax ->
// P V.  One barrier per tile says "all products of this tile so far are done" (S of block j and, before it, P V of block
// j - 1), so the softmax may overwrite S with P and rescale O without another wait.  What bounds the kernel now is that
// chain: per block of 128 keys an SM spends 3900 clocks on both tiles, the starts and ends of its CTAs included; the tensor core
// is busy for 2050 of them (its counter: 50 %) and the special-function units, which the two warpgroups share, for 2050 too (52 %):
// the softmax of a tile, its products and the hand-over follow one another, and two tiles are not enough to fill the gaps of
// both.  Measured at 32 heads x 4096 x 128 bf16, before -> after: causal 174 -> 139 us (990 TFLOP/s), full 300 -> 255 us;
// 32 heads x 16384 causal 1790 us (1230 TFLOP/s).  Tried and not kept: a quarter to a half of the exponentials as polynomials
// on the FMA pipe (+2 to +10 % time), two warpgroups per tile (+11 %), S in halves of 64 keys issued ahead (+12 %: an N64
// product is bound by reading A from shared memory).
// The exponent's reference maximum m is only raised when the running maximum has grown by more than 2^8 ("lazy"
// rescaling): then the warpgroup multiplies its rows of O in TMEM (tcgen05.ld / st) before it releases P.  That is rare
// after the first blocks, so O normally never leaves TMEM until the epilogue.
// The MMA warp alternates between the tiles (P V and next S of tile 0, then of tile 1), so one tile's softmax runs while
// the tensor core works for the other; K and V tiles stream through a five-slot TMA ring.
//
// kWin (sliding window of W keys and s sinks): the blocks without a visible key are left out.  The list of blocks that the two
// tiles share is, in this order: the blocks that only tile 0's window reaches (one, or none), the blocks of the sinks, the
// rest of tile 1's window.  So tile 0 takes a prefix of the list and tile 1 a suffix, and every block is loaded once.  Packed
// rows of the next sequence, or of nobody, are set to zero in the last block of V: their probability is zero, but zero times
// what lies there need not be.  Measured: 32 heads x 4096, window 1024: 88 us (680 TFLOP/s of what is visible, tensor core
// 39 % busy; 96 us with a CTA per unit); one prompt of 8192, window 4096: 352 us (1170 TFLOP/s, 56 %).
// One unit of work: a pair of query tiles of one (batch, head); heavy (late) tiles first, across all (batch, head) instances, or within each
// sequence where they are packed and windowed.
struct FwdUnit {
  int qp, b, h, hk, Sq, Sk, qoff, koff, bt;
  int nb0, nb1, nbmax;        // tile t ends before item nb<t> of the list of key blocks
  __device__ __forceinline__ int nb(int t) const { return t ? nb1 : nb0; }
  // kWin: the list that the tiles share is [lo0, lo0 + n_pre), then the sinks' [0, n_sink), then [lo1, ...); tile 1 begins at item
  // second_first
  int second_first, lo0, lo1, n_pre, n_sink;
};

template <typename T, bool kWin>
__global__ void __launch_bounds__(kAttnThreads, 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                const __grid_constant__ CUtensorMap tmap_v, T* __restrict__ out, const AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;                          // [2][kTile]
  uint8_t* sR = smem + 2 * kTile;              // [kRing][kTile]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (2 + kRing) * kTile);
  uint64_t* q_full = bars;                     // [2]
  uint64_t* r_full = bars + 2;                 // [kRing]
  uint64_t* r_empty = bars + 2 + kRing;        // [kRing]  tcgen05.commit
  uint64_t* mma_done = bars + 2 + 2 * kRing;   // [2]      tcgen05.commit: P V of block j - 1 and S of block j
  uint64_t* p_ready = mma_done + 2;            // [2][2]   four softmax warps: first / second part of P of block j is in TMEM
  uint64_t* q_empty = p_ready + 4;             // [2]      tcgen05.commit: the last S of a unit's tile (kWin)
  uint64_t* u_full = q_empty + 2;              // [2]      a unit's description is there (kWin)
  uint64_t* u_empty = u_full + 2;              // [2]      all have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(u_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  FwdUnit* s_unit = reinterpret_cast<FwdUnit*>(tmem_slot + 2);      // [2]
  static_assert(24 * 8 + 8 + 2 * sizeof(FwdUnit) <= 512, "barriers and units share 512 bytes");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_bh = p.B * p.H;
  auto complete = [&](FwdUnit& u) {      // from qp, b and h
    u.hk = u.h / (p.H / p.Hkv);
    // this instance's sequence: lengths, first packed rows and the batch coordinate of the tensor maps.  Rows past a
    // packed sequence's end belong to the next sequence: they are loaded, masked by index and never stored.
    u.Sq = p.Sq;
    u.Sk = p.Sk;
    u.bt = u.b;
    if (p.cu_q) {
      u.qoff = p.cu_q[u.b];
      u.Sq = p.cu_q[u.b + 1] - u.qoff;
      u.koff = p.cu_k[u.b];
      u.Sk = p.cu_k[u.b + 1] - u.koff;
      u.bt = 0;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int q0 = (2 * u.qp + t) * AQ;
      int k_end = u.Sk;
      if (p.causal) k_end = min(u.Sk, q0 + AQ);
      (t ? u.nb1 : u.nb0) = q0 < u.Sq ? (k_end + AK - 1) / AK : 0;
    }
    if constexpr (kWin) {
      const int sb = (min(p.sinks, u.Sk) + AK - 1) / AK, q0 = 2 * u.qp * AQ;
      const bool second = q0 + AQ < u.Sq;
      u.lo0 = max(max(0, q0 - p.window + 1) / AK, sb);
      u.lo1 = second ? max(max(0, q0 + AQ - p.window + 1) / AK, sb) : u.lo0;
      const int end0 = u.nb0, end1 = u.nb1;
      u.n_pre = max(0, min(u.lo1, end0) - u.lo0);
      u.n_sink = min(sb, max(end0, end1));
      u.nb0 = u.n_pre + min(sb, end0) + max(0, end0 - u.lo1);
      u.nb1 = second ? u.n_pre + u.n_sink + max(0, end1 - u.lo1) : 0;
      if (u.nb1 == u.n_pre) u.nb1 = 0;      // no key at all
      u.second_first = u.nb1 > 0 ? u.n_pre : 0;
    }
    u.nbmax = max(u.nb0, u.nb1);
  };
  auto make_unit = [&](int unit) {
    FwdUnit u{};
    u.qp = p.q_pairs - 1 - unit / n_bh;
    const int bh = unit % n_bh;
    u.b = bh / p.H;
    u.h = bh - u.b * p.H;
    complete(u);
    return u;
  };
  // Calls f() for every unit of this CTA until it returns false.  Without a window a CTA has one unit.  With one the units are short (ten
  // blocks at a window of 1024): a CTA then stays on its SM and takes every 148th unit, turning round at either end so that long and
  // short ones even out; the loads and the first products of a unit run while the one before it is stored.  A warp of its own finds the
  // units, two ahead, and hands them over: each role for itself would pay for the search in time and in registers.
  const FwdUnit only = kWin ? FwdUnit{} : make_unit((int)blockIdx.x);
  auto each_unit = [&](auto whole_warp, auto f) {
    if constexpr (!kWin) {
      f(only);
    } else {
      for (uint32_t n = 0;; ++n) {
        if constexpr (decltype(whole_warp)::value) {
          if (!mbar_wait_warp(&u_full[n & 1], (n >> 1) & 1, abort_flag)) break;
        } else {
          if (!mbar_wait(&u_full[n & 1], (n >> 1) & 1, abort_flag)) break;
        }
        const FwdUnit u = s_unit[n & 1];
        if constexpr (decltype(whole_warp)::value) __syncwarp();
        if (!decltype(whole_warp)::value || lane == 0) mbar_arrive(&u_empty[n & 1]);
        if (u.qp < 0 || !f(u)) break;
      }
    }
  };
  auto first_of = [](const FwdUnit& u, int t) { return kWin && t == 1 ? u.second_first : 0; };
  auto block_of = [](const FwdUnit& u, int j) {
    if constexpr (!kWin) return j;
    else return j < u.n_pre ? u.lo0 + j : (j - u.n_pre < u.n_sink ? j - u.n_pre : u.lo1 + (j - u.n_pre - u.n_sink));
  };

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&u_full[t], 1);
      mbar_init(&u_empty[t], kUnitReaders);
      mbar_init(&mma_done[t], 1);
      mbar_init(&p_ready[2 * t], 4);
      mbar_init(&p_ready[2 * t + 1], 4);
    }
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&r_full[s], 1);
      mbar_init(&r_empty[s], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, kAttnTmemCols);
    tmem_relinquish();
  }
  auto tile_pairs = [&](int b) { return min(p.q_pairs, (max(0, p.cu_q[b + 1] - p.cu_q[b]) + 2 * AQ - 1) / (2 * AQ)); };
  UnitWalk walk;
  if (kWin && warp == 10 && p.cu_q) walk.take(0, 0, p.B, lane, tile_pairs);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp >= 8) {
    regs_dec<kOtherRegs>();
    if (warp == 8) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        int ring = 0;                    // items of the ring so far
        uint32_t loaded[2] = {0, 0};     // Q tiles so far, for the phases
        each_unit(std::false_type{}, [&](const FwdUnit& u) -> bool {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (u.nb(t) == 0) continue;
            const int q0 = (2 * u.qp + t) * AQ;
            if (kWin && !mbar_wait(&q_empty[t], (loaded[t] & 1) ^ 1, abort_flag)) return false;
            ++loaded[t];
            mbar_expect_tx(&q_full[t], kTile);
            tma_load_4d(sQ + t * kTile, &tmap_q, &q_full[t], 0, u.qoff + q0, u.h, u.bt);                 // d 0..63
            tma_load_4d(sQ + t * kTile + kTile / 2, &tmap_q, &q_full[t], 64, u.qoff + q0, u.h, u.bt);    // d 64..127
          }
          for (int n = 0; n < 2 * u.nbmax; ++n, ++ring) {
            const int st = ring % kRing;
            if (!mbar_wait(&r_empty[st], (uint32_t)(((ring / kRing) & 1) ^ 1), abort_flag)) return false;
            mbar_expect_tx(&r_full[st], kTile);
            const int k0 = block_of(u, n >> 1) * AK;
            const CUtensorMap* map = (n & 1) ? &tmap_v : &tmap_k;   // V is read as an MN-major B operand: same boxes
            tma_load_4d(sR + st * kTile, map, &r_full[st], 0, u.koff + k0, u.hk, u.bt);
            tma_load_4d(sR + st * kTile + kTile / 2, map, &r_full[st], 64, u.koff + k0, u.hk, u.bt);
          }
          return true;
        });
      }
      __syncwarp();
    } else if (warp == 9) {
      // ------------------------------------------------------------ MMA issuer (the whole warp waits, one lane issues)
      // instruction descriptors: fp32 accumulate, bf16/fp16 operands, M128 N128; S: both K-major; PV: B MN-major
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      constexpr uint32_t idesc_o = idesc_s | (1u << 16);
      const bool leader = elect_one();
      const uint64_t q_desc = make_desc(smem_u32(sQ), 16, 1024);             // K-major tiles; + (bytes >> 4) for an offset
      const uint64_t k_desc = make_desc(smem_u32(sR), 16, 1024);
      const uint64_t v_desc = make_desc(smem_u32(sR), kTile / 2, 1024);      // MN-major
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_warp(bar, parity, abort_flag); };
      auto ring_wait = [&](int n) { return wait(&r_full[n % kRing], (uint32_t)((n / kRing) & 1)); };
      auto issue_s = [&](int t, int n) {     // S_t = Q_t K^T with K in ring item n
        const uint64_t qa = q_desc + (uint32_t)(t * (kTile >> 4)), ka = k_desc + (uint32_t)((n % kRing) * (kTile >> 4));
  #pragma unroll
        for (int kk = 0; kk < AD / 16; ++kk) {
          const uint32_t off = ((uint32_t)(kk >> 2) * (kTile / 2) + (uint32_t)(kk & 3) * 32) >> 4;   // 64-column atom, 32 B per k16
          umma_f16(tmem_base + (uint32_t)(t * 128), qa + off, ka + off, idesc_s, kk != 0 ? 1u : 0u);
        }
      };
      auto issue_pv = [&](int t, int n, bool first, int kk0, int kk1) {   // O_t (+)= P_t V with V in ring item n
        const uint32_t pa = tmem_base + (uint32_t)(t * 128);
        const uint64_t va = v_desc + (uint32_t)((n % kRing) * (kTile >> 4));
  #pragma unroll
        for (int kk = kk0; kk < kk1; ++kk)
          // A = P in TMEM, 8 columns per 16 keys; B = V (MN-major): 16 key rows = 2048 B, next 64-wide d box 16 KB on
          umma_f16_ts(tmem_base + 256u + (uint32_t)(t * 128), pa + (uint32_t)(kk * 8), va + (uint32_t)(kk * (2048 >> 4)), idesc_o,
                      (first && kk == 0) ? 0u : 1u);
      };
      int ring = 0;                      // items of the ring before this unit's
      uint32_t q_seen[2] = {0, 0}, p_seen[2] = {0, 0};     // Q tiles and blocks of P so far, for the phases
      each_unit(std::true_type{}, [&](const FwdUnit& u) -> bool {
        bool ok = true;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (u.nb(t) > 0 && ok) ok = wait(&q_full[t], kWin ? q_seen[t]++ & 1 : 0u);
        if (ok && u.nbmax > 0) ok = ring_wait(ring);
        if (ok && u.nbmax > 0) {
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (u.nb(t) > 0 && first_of(u, t) == 0) {
                issue_s(t, ring);
                if (kWin && u.nb(t) == 1) umma_commit(&q_empty[t]);
                umma_commit(&mma_done[t]);
              }
            umma_commit(&r_empty[ring % kRing]);
          }
        }
        for (int j = 0; j < u.nbmax && ok; ++j) {
          const int nv = ring + 2 * j + 1, nk = ring + 2 * j + 2;
          if (!ring_wait(nv)) { ok = false; break; }
          if (j + 1 < u.nbmax && !ring_wait(nk)) { ok = false; break; }
          if constexpr (kWin) {
            const int rows = u.Sk - block_of(u, j) * AK;      // of this block that are the sequence's own
            if (p.cu_q && rows < AK) {
              uint8_t* tile = sR + (nv % kRing) * kTile;
              for (int x = rows * 8 + lane; x < AK * 8; x += 32) {
                *reinterpret_cast<uint4*>(tile + x * 16) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(tile + kTile / 2 + x * 16) = make_uint4(0, 0, 0, 0);
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
            }
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int j0 = first_of(u, t);
            const bool next = j + 1 < u.nb(t) && j + 1 >= j0, last = kWin && j + 2 == u.nb(t);
            if (j >= u.nb(t) || !ok) continue;
            if (j < j0) {
              if (next && leader) {
                issue_s(t, nk);
                if (last) umma_commit(&q_empty[t]);
                umma_commit(&mma_done[t]);
              }
              continue;
            }
            const uint32_t par = kWin ? p_seen[t]++ & 1 : (uint32_t)(j & 1);
            if (!wait(&p_ready[2 * t], par)) { ok = false; continue; }
            tc_fence_after();
            if (leader) issue_pv(t, nv, j == j0, 0, kFirstPart / 16);
            if (!wait(&p_ready[2 * t + 1], par)) { ok = false; continue; }
            tc_fence_after();
            if (leader) {
              issue_pv(t, nv, false, kFirstPart / 16, AK / 16);
              if (next) {
                issue_s(t, nk);              // over P of block j: the tensor core works in issue order
                if (last) umma_commit(&q_empty[t]);
              }
              umma_commit(&mma_done[t]);
            }
          }
          if (!ok) break;
          if (leader) {
            umma_commit(&r_empty[nv % kRing]);
            if (j + 1 < u.nbmax) umma_commit(&r_empty[nk % kRing]);
          }
        }
        ring += 2 * u.nbmax;
        return ok;
      });
      __syncwarp();
    } else if (kWin && warp == 10) {
      // ------------------------------------------------------------ the units, one after the other; qp < 0 behind the last
      for (uint32_t n = 0;; ++n) {
        const int unit = (int)(n * gridDim.x + (n & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x));
        FwdUnit u{};
        bool there;
        if (p.cu_q) {
          int behind;
          there = walk.find(unit / p.H, p.B, lane, u.b, behind, tile_pairs);
          if (there) {
            u.h = unit % p.H;
            u.qp = tile_pairs(u.b) - 1 - behind;
            complete(u);
          }
        } else {
          there = unit < p.units;
          if (there) u = make_unit(unit);
        }
        if (!there) u.qp = -1;
        if (!mbar_wait_warp(&u_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag)) break;
        if (lane == 0) {
          s_unit[n & 1] = u;
          mbar_arrive(&u_full[n & 1]);
        }
        __syncwarp();
        if (!there) break;
      }
    }
  } else {
    regs_inc<kSoftmaxRegs>();
    // ------------------------------------------------------------ softmax warpgroup t (warps 4t .. 4t+3)
    const int t = warp >> 2;
    const int qw = warp & 3;                 // TMEM lane quarter of this warp
    const int r = qw * 32 + lane;            // query row inside the tile = TMEM lane
    const uint32_t lane_base = ((uint32_t)(qw * 32) << 16);
    const uint32_t s_addr = tmem_base + lane_base + (uint32_t)(t * 128);
    const uint32_t o_addr = tmem_base + lane_base + 256u + (uint32_t)(t * 128);
    // warp-uniform wait: the warp-collective TMEM accesses and votes below need all 32 lanes to take the same path
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
      const bool w = mbar_wait(bar, parity, abort_flag);
      return __all_sync(0xffffffffu, w);
    };
    T* const rest = kWin ? (T*)p.remainder : nullptr;
    uint32_t done = 0;                       // phases of mma_done[t] so far
    each_unit(std::true_type{}, [&](const FwdUnit& u) -> bool {
      const int qi = (2 * u.qp + t) * AQ + r;
      float m_ref = -INFINITY;                 // maximum the exponents refer to (raised lazily)
      float l_run = 0.f;
      bool ok = true;
      const int n_blocks = u.nb(t) - first_of(u, t);
      for (int j = 0; j < n_blocks; ++j) {
        if (!wait_all(&mma_done[t], kWin ? done++ & 1 : (uint32_t)(j & 1))) { ok = false; break; }
        tc_fence_after();
        const int k0 = block_of(u, j + first_of(u, t)) * AK;
        // the row's visible keys: [0, lim), without [hide0, hide1) in front of the window
        int lim = u.Sk - k0;
        if (p.causal) lim = min(lim, qi - k0 + 1);
        lim = max(0, min(lim, AK));
        const int hide0 = kWin ? max(0, p.sinks - k0) : 0, hide1 = kWin ? qi - p.window + 1 - k0 : 0;
        const bool full = __all_sync(0xffffffffu, lim == AK && hide0 >= hide1);
        // the whole row of scores in registers
        uint32_t raw[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + (uint32_t)(c * 32), raw[c]);
        tmem_ld_wait();
        // kWin: what the row does not see becomes -inf here, two instructions an element, and the block goes the common way.  The tests
        // inside the loops below, three times for each element, are four times the code, and a windowed CTA meets a masked block so
        // often that it waits for instructions: 32 heads x 4096, window 64, 174 us with them.
        if constexpr (kWin) {
          if (!full) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t seen = low_bits(lim - c * 32) & ~(low_bits(hide1 - c * 32) & ~low_bits(hide0 - c * 32));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((seen >> e) & 1u)) raw[c][e] = 0xff800000u;
            }
          }
        }
        // P = exp2(S * scale - m) as bf16 / fp16 pairs over the first 64 columns of S; packed fp32 arithmetic, one
        // special-function instruction per exponential, one conversion per pair.  Two instantiations: with the mask test
        // inside one, every element pays a compare and a select.
        float l0, l1;
        uint32_t pk[4][16];
        auto chunk_p = [&](auto masked, int c, float neg_m) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x0, x1;
            fma2(x0, x1, __uint_as_float(raw[c][e]), __uint_as_float(raw[c][e + 1]), p.scale_log2, neg_m);
            float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            if constexpr (decltype(masked)::value) {
              if (c * 32 + e >= lim) p0 = 0.f;
              if (c * 32 + e + 1 >= lim) p1 = 0.f;
            }
            add2(l0, l1, p0, p1);
            pk[c][e >> 1] = pack2<T>(p0, p1);
          }
        };
        auto block = [&](auto masked) {
          // The first part is computed against the reference maximum as it stands, while the block's own maximum is found
          // beside it (four chains of three-input maxima under the special-function unit's shadow): m is raised in the first
          // block and hardly ever after it, and only then is the first part computed again.
          l0 = l1 = 0.f;
          const float m_old = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll
          for (int c = 0; c < kFirstPart / 32; ++c) chunk_p(masked, c, -m_old);
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float a = __uint_as_float(raw[c][e]), b2 = __uint_as_float(raw[c][e + 1]);
              if constexpr (decltype(masked)::value) {
                if (c * 32 + e >= lim) a = -INFINITY;
                if (c * 32 + e + 1 >= lim) b2 = -INFINITY;
              }
              mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], a, b2);
            }
          const float m_blk = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const float m_new = fmaxf(m_ref, m_blk * p.scale_log2);
          const bool raise = m_new - m_ref > kRescaleThreshold;      // also true for the first finite maximum
          if (__any_sync(0xffffffffu, raise)) {
            const float alpha = raise ? exp2f(m_ref - m_new) : 1.f;   // 0 when m_ref = -inf
            if (j > 0) {
#pragma unroll
              for (int c = 0; c < AD / 16; ++c) {
                uint32_t o16[16];
                tmem_ld16(o_addr + (uint32_t)(c * 16), o16);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o16[e] = __float_as_uint(__uint_as_float(o16[e]) * alpha);
                tmem_st16(o_addr + (uint32_t)(c * 16), o16);
              }
            }
            if (raise) {
              l_run *= alpha;
              m_ref = m_new;
            }
            l0 = l1 = 0.f;
            const float m_use = m_ref == -INFINITY ? 0.f : m_ref;     // row without any visible key so far
#pragma unroll
            for (int c = 0; c < kFirstPart / 32; ++c) chunk_p(masked, c, -m_use);
          }
#pragma unroll
          for (int c = 0; c < kFirstPart / 32; ++c) tmem_st16(s_addr + (uint32_t)(c * 16), pk[c]);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[2 * t]);
          const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll
          for (int c = kFirstPart / 32; c < 4; ++c) {
            chunk_p(masked, c, -m_use);
            tmem_st16(s_addr + (uint32_t)(c * 16), pk[c]);
          }
        };
        if constexpr (kWin) {
          block(std::false_type{});
        } else {
          if (full) block(std::false_type{});
          else block(std::true_type{});
        }
        l_run += l0 + l1;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[2 * t + 1]);
      }
      if (ok && n_blocks > 0) ok = wait_all(&mma_done[t], kWin ? done++ & 1 : (uint32_t)(n_blocks & 1));
      if (ok && n_blocks > 0) {
        tc_fence_after();
        const float inv = l_run > 0.f ? 1.f / l_run : 0.f;
        const int64_t at = (int64_t)u.bt * p.o_sb + (int64_t)u.h * p.o_sh + (int64_t)(u.qoff + qi) * p.o_ss;
        T* orow = out + at;
        auto store = [&](auto both) {      // with the remainder: two stores of 32 bytes (91 us for 32 heads x 4096, window 1024; 104 with four of 16)
#pragma unroll
          for (int c = 0; c < AD / 32; ++c) {
            uint32_t raw[32];
            tmem_ld32(o_addr + (uint32_t)(c * 32), raw);
            tmem_ld_wait();
            if (qi >= u.Sq) continue;
            if constexpr (decltype(both)::value) {
#pragma unroll
              for (int g16 = 0; g16 < 2; ++g16) {
                uint32_t v[8], w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const float x0 = __uint_as_float(raw[g16 * 16 + 2 * e]) * inv, x1 = __uint_as_float(raw[g16 * 16 + 2 * e + 1]) * inv;
                  v[e] = pack2<T>(x0, x1);
                  const float2 r2 = unpack2<T>(v[e]);
                  w[e] = pack2<T>(x0 - r2.x, x1 - r2.y);
                }
                st32(orow + c * 32 + g16 * 16, v);
                st32(rest + at + c * 32 + g16 * 16, w);
              }
            } else {
#pragma unroll
              for (int g8 = 0; g8 < 4; ++g8) {
                Vec16<T> v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v.v[e] = ToF<T>::from(__uint_as_float(raw[g8 * 8 + e]) * inv);
                st16(orow + c * 32 + g8 * 8, v);
              }
            }
          }
        };
        if constexpr (kWin) {
          if (rest) store(std::true_type{});
          else store(std::false_type{});
        } else {
          store(std::false_type{});
        }
        if (qi < u.Sq && p.lse)
          p.lse[p.cu_q ? (int64_t)u.h * p.total_q + u.qoff + qi : ((int64_t)u.b * p.H + u.h) * p.Sq + qi] =
              l_run > 0.f ? (m_ref + log2f(l_run)) * 0.6931471805599453f : -INFINITY;
      }
      if constexpr (kWin) {
        Vec16<T> zero;
#pragma unroll
        for (int e = 0; e < 8; ++e) zero.v[e] = ToF<T>::from(0.f);
        if (n_blocks == 0 && qi < u.Sq) {                  // a query that sees no key
          const int64_t at = (int64_t)u.bt * p.o_sb + (int64_t)u.h * p.o_sh + (int64_t)(u.qoff + qi) * p.o_ss;
          for (int c = 0; c < AD; c += 8) {
            st16(out + at + c, zero);
            if (rest) st16(rest + at + c, zero);
          }
          if (p.lse) p.lse[p.cu_q ? (int64_t)u.h * p.total_q + u.qoff + qi : ((int64_t)u.b * p.H + u.h) * p.Sq + qi] = -INFINITY;
        }
      }
      return ok;
    });
    if constexpr (kWin) {
      if (p.cu_q) {                                    // packed rows past the last sequence: zeros, the CTAs share them
        Vec16<T> zero;
#pragma unroll
        for (int e = 0; e < 8; ++e) zero.v[e] = ToF<T>::from(0.f);
        for (int x = p.cu_q[p.B] + blockIdx.x * 16 + (threadIdx.x >> 4); x < p.total_q; x += gridDim.x * 16)
          for (int y = 0; y < p.H; ++y) {
            const int64_t at = (int64_t)y * p.o_sh + (int64_t)x * p.o_ss + (threadIdx.x & 15) * 8;
            st16(out + at, zero);
            if (rest) st16(rest + at, zero);
            if (p.lse && (threadIdx.x & 15) == 0) p.lse[(int64_t)y * p.total_q + x] = -INFINITY;
          }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kAttnTmemCols);
  }
  settle_abort(abort_flag, p.status);
}

template <typename K>
int fwd_setup(K kern) {
  cudaFuncAttributes at;
  cudaError_t e = cudaFuncGetAttributes(&at, kern);
  if (e != cudaSuccess) return (int)e;
  if (at.numRegs < kLaunchRegs) return (int)cudaErrorNotSupported;   // the register split would wait for ever
  return opt_in_smem(kern, kAttnSmem);
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int b200_flash_attn_fwd(const b200_attn_t* a, void* out, float* lse, const void* q, const void* k,
                                   const void* v, cudaStream_t stream) {
  if (a->head_dim != AD || (a->dtype != B200_BF16 && a->dtype != B200_F16) || a->B <= 0 || a->H <= 0 || a->Hkv <= 0 ||
      a->H % a->Hkv != 0 || a->Sq <= 0 || a->Sk <= 0)
    return (int)cudaErrorNotSupported;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  auto st_ok = [](int64_t s) { return s % 8 == 0; };
  if (!al(q) || !al(k) || !al(v) || !al(out) || !st_ok(a->q_sb) || !st_ok(a->q_sh) || !st_ok(a->q_ss) || !st_ok(a->k_sb) ||
      !st_ok(a->k_sh) || !st_ok(a->k_ss) || !st_ok(a->v_sb) || !st_ok(a->v_sh) || !st_ok(a->v_ss) || !st_ok(a->o_sb) ||
      !st_ok(a->o_sh) || !st_ok(a->o_ss))
    return (int)cudaErrorNotSupported;
  // a broadcast (zero) stride cannot be a tensor-map stride
  if ((a->B > 1 && !a->cu_seqlens_q && (a->q_sb == 0 || a->k_sb == 0 || a->v_sb == 0)) || (a->H > 1 && a->q_sh == 0) ||
      (a->Hkv > 1 && (a->k_sh == 0 || a->v_sh == 0)) || a->q_ss == 0 || a->k_ss == 0 || a->v_ss == 0)
    return (int)cudaErrorNotSupported;
  const int bf16 = a->dtype == B200_BF16;
  CUtensorMap mq, mk, mv;
  auto nz = [](int64_t s, int64_t fallback) { return s ? s : fallback; };
  const bool packed = a->cu_seqlens_q != nullptr;
  if (packed) {
    if (!a->cu_seqlens_k || a->total_q <= 0 || a->total_k <= 0) return (int)cudaErrorNotSupported;
    // one "batch" of total rows: the kernel adds each sequence's first row to its tile coordinates
    if (!make_attn_map(&mq, q, bf16, 1, a->H, a->total_q, (int64_t)a->total_q * a->q_ss, nz(a->q_sh, 8), a->q_ss) ||
        !make_attn_map(&mk, k, bf16, 1, a->Hkv, a->total_k, (int64_t)a->total_k * a->k_ss, nz(a->k_sh, 8), a->k_ss) ||
        !make_attn_map(&mv, v, bf16, 1, a->Hkv, a->total_k, (int64_t)a->total_k * a->v_ss, nz(a->v_sh, 8), a->v_ss))
      return (int)cudaErrorNotSupported;
  } else if (!make_attn_map(&mq, q, bf16, a->B, a->H, a->Sq, nz(a->q_sb, 8), nz(a->q_sh, 8), a->q_ss) ||
             !make_attn_map(&mk, k, bf16, a->B, a->Hkv, a->Sk, nz(a->k_sb, 8), nz(a->k_sh, 8), a->k_ss) ||
             !make_attn_map(&mv, v, bf16, a->B, a->Hkv, a->Sk, nz(a->v_sb, 8), nz(a->v_sh, 8), a->v_ss))
    return (int)cudaErrorNotSupported;
  AttnParams p{};
  p.B = a->B; p.H = a->H; p.Hkv = a->Hkv; p.Sq = a->Sq; p.Sk = a->Sk;
  p.causal = a->causal;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.o_sb = a->o_sb; p.o_sh = a->o_sh; p.o_ss = a->o_ss;
  p.lse = lse;
  p.cu_q = a->cu_seqlens_q;
  p.cu_k = a->cu_seqlens_k;
  p.total_q = a->total_q;
  p.q_blocks = (a->Sq + AQ - 1) / AQ;
  p.q_pairs = (p.q_blocks + 1) / 2;
  p.status = gemm_status_word_device();
  const long long grid = (long long)a->B * a->H * p.q_pairs;
  if (grid > 2147483647ll - 1024) return (int)cudaErrorNotSupported;
  p.units = (int)grid;
  p.remainder = a->remainder;
  p.window = a->window;
  p.sinks = a->sinks;
  auto launch = [&](auto kern, OncePerDevice& once, auto* o) -> int {
    if (int e = once([&] { return fwd_setup(kern); })) return e;
    const unsigned ctas = a->window > 0 ? (unsigned)std::min<long long>(grid, gemm_sm_count()) : (unsigned)grid;
    kern<<<ctas, kAttnThreads, kAttnSmem, stream>>>(mq, mk, mv, o, p);
    B200K_LAUNCH_RET();
  };
  static OncePerDevice once[4];
  if (a->window > 0) {
    if (!a->causal || a->window > (1 << 30) || a->sinks < 0) return (int)cudaErrorNotSupported;
    if (a->remainder && (((reinterpret_cast<uintptr_t>(a->remainder) | reinterpret_cast<uintptr_t>(out)) & 31) || a->o_sb % 16 || a->o_sh % 16 || a->o_ss % 16))
      return (int)cudaErrorNotSupported;                                                     // stored 32 bytes at a time
    return bf16 ? launch(attn_fwd_kernel<__nv_bfloat16, true>, once[2], (__nv_bfloat16*)out)
                : launch(attn_fwd_kernel<__half, true>, once[3], (__half*)out);
  }
  return bf16 ? launch(attn_fwd_kernel<__nv_bfloat16, false>, once[0], (__nv_bfloat16*)out)
              : launch(attn_fwd_kernel<__half, false>, once[1], (__half*)out);
}
