// Flash-attention backward under a sliding window with sinks (head_dim 128, bf16 / fp16, grouped-query heads): key j is visible to query i
// when j <= i and (i - j < window or j < sinks).
//
// The products, the layouts and the roles of the warps are those of attention_bwd.cu, whose comment has them: everything is computed
// transposed, keys along the TMEM lanes; dK and dV accumulate in TMEM over the query blocks of a unit, dQ leaves by TMA reductions into
// fp32.  What differs:
//   * The queries that see a block of keys are a contiguous range, window + 127 long behind the block's first key, or all that follow when
//     it holds sinks.  A block with sinks meets many more query blocks than the others (at 4096 tokens and a window of 1024: 32 against
//     9, times the heads of a group), so its range is cut into chunks of about the others' length, in each sequence by its own length;
//     their dV and dK go to fp32 buffers that a small kernel adds up in order.
//   * Units are short, and starting and ending a CTA cost as much as three or four pairs of blocks: a CTA stays on its SM and takes every
//     148th unit, turning round at either end so that long and short ones even out.  The loads of a unit's queries, and the waits for its
//     first products, run while the one before it is stored.  A warp of its own finds the units and hands them over.  What a change of
//     units still costs, about 5 us of 27 for nine pairs, is the chain K -> S^T -> P -> dS that starts afresh: K and V of the next unit have
//     no place before the last product of this one.
//   * Hidden scores become -inf before the exponentials, two instructions an element, instead of tests inside the loops, whose second
//     copy of the code cost more than they did (instructions came late).
//   * The row sums of dO O are taken with what rounding left of O, which the forward keeps for it: with few keys in a window dS is a
//     difference of nearly equal numbers, and the rounded O alone put the gradients of q and k off by 3.7e-3 of their norm (two keys, bf16),
//     now 2.5e-3 as with many keys: dS is rounded before its products (1.7e-3, as much as the result's own rounding).  It costs 4.5 % of
//     forward and backward at a window of 1024 (348 -> 364 us, 32 heads x 4096), 6 % at 256 and below.
//   * dS goes into its products without the softmax scale, which dQ and dK get in 32 bits when they leave TMEM: in fp16 its values are small
//     under a long window, and a scale of 0.088 in front of the rounding would take three and a half bits more from them (4096 keys, dO of
//     2^-10: dQ and dK off by 1.3e-2 of their norm with it, 1.2e-3 without).  In return fp16's largest value, 65504, bounds P (dP - delta)
//     itself and not 0.088 of it.
//   * Packed rows that are not the sequence's own are zeros in shared memory before a product reads them: their probabilities are zero,
//     but zero times what lies there need not be.
// Measured (whole calls: row dots, this kernel, sums of the chunks, conversion of dQ): 32 heads x 4096, window 1024, four sinks 277 us
// (247 without sinks; a CTA per unit took 15 more); with 8 key heads 269 us.  Tried and not kept: cutting the list of pairs into 148 equal
// shares, so that units are cut anywhere (32 heads x 4096: 484 us; neighbouring CTAs no longer read the same rows, and twice as many
// units begin afresh).
//
// Parity: no counterpart in the reference (its vendor flash backward takes a causal flag only: reference
// torch_musa/csrc/aten/ops/attention/mudnn/SDP.cpp:678-845).
#include "attention_bwd_common.cuh"

#include <algorithm>
#include <type_traits>

namespace b200k {
namespace {
using namespace gemmdev;
using namespace attndev;

struct WindowParams {
  int B, H, Hkv, Sq, Sk;
  float scale, scale_log2;      // of dQ and dK; of the exponents, times log2(e)
  const float* lse;       // [B, H, Sq] natural log
  const float* delta;     // [B, H, Sq]
  float* dq;              // [B, H, Sq, 128] fp32
  int64_t dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int kv_blocks, q_blocks;
  int* status;
  // packed variable-length sequences (NULL: dense batch), as in the forward kernel; lse / delta are then [H, total_q]
  // and dq [H, total_q, 128]
  const int* cu_q;
  const int* cu_k;
  int total_q;
  int window, sinks, total_k;
  int units;                      // units of work that the CTAs share
  int sink_blocks, sink_chunk;    // key blocks with sinks (of a long sequence), query blocks of a chunk of theirs
  int sink_slots;                 // places of chunks; 0: no sequence has more than one
  float* sink_ws;                 // fp32 [sink_slots][sink_blocks][Hkv][dV, dK][128][128]
};

// Query blocks of sequence b, and the chunks into which those of its sinks are cut.
__device__ __forceinline__ int query_blocks(const WindowParams& p, int b) {
  return p.cu_q ? min(p.q_blocks, (max(0, p.cu_q[b + 1] - p.cu_q[b]) + BQ - 1) / BQ) : p.q_blocks;
}
__device__ __forceinline__ int chunks_of(const WindowParams& p, int q_blocks) { return max(1, (q_blocks + p.sink_chunk - 1) / p.sink_chunk); }
// The first of sequence b's places.  Packed sequences find theirs by their first row alone, without a sum over those in front: with
// c = sink_chunk, n > c query blocks are at least 128 (n - 1) + 1 rows and n' = ceil(n / c) = floor((n - 1) / c) + 1 chunks, so that
// n' <= 2 floor((n - 1) / c) <= 2 rows / (128 c), and ceil(x + y) - ceil(x) >= floor(y).
__host__ __device__ __forceinline__ int slots_before(int rows, int chunk) {
  const unsigned c = BQ / 2 * (unsigned)chunk;
  return (int)(((unsigned)rows + c - 1) / c);
}
__device__ __forceinline__ int first_slot(const WindowParams& p, int b) {
  return p.cu_q ? slots_before(p.cu_q[b], p.sink_chunk) : b * chunks_of(p, p.q_blocks);
}

// The query blocks [first, end) that see key block kb.
__device__ __forceinline__ void window_queries(const WindowParams& p, int kb, int Sq, int Sk, int q_blocks, int& first, int& end) {
  const int k0 = kb * BK;
  first = min(q_blocks, k0 / BQ);
  end = k0 < p.sinks ? q_blocks : min(q_blocks, (min(k0 + BK, Sk) - 1 + p.window - 1) / BQ + 1);
  if (k0 >= Sk || end < first) end = first;
}

// Rows [rows, 128) of a tile that a copy brought into shared memory become zero (called by a converged warp, before its products
// read the tile): they belong to another sequence, or to nobody.
__device__ __forceinline__ void zero_tail(uint8_t* tile, int rows, int lane) {
  for (int x = rows * 8 + lane; x < 128 * 8; x += 32) {
    *reinterpret_cast<uint4*>(tile + x * 16) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(tile + kTile / 2 + x * 16) = make_uint4(0, 0, 0, 0);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

constexpr int kUnitReaders = 15;         // every other warp of the kernel
constexpr int kUnitBytes = 128;          // of their descriptions, beyond the common layout's: from the slack

// One unit of work: a key block of one (batch, kv head), or a chunk of one.  All (batch, head) instances of the earliest key block come
// first (under a causal mask it meets the most query blocks); of packed sequences all that hold sinks.
struct BwdUnit {
  int kb, chunk, bh, b, hk, k0, Sq, Sk, qoff, koff, bt;
  int i0, n_i, n_it, h0, istart;      // first query block, query blocks, pairs of query block and head, where the pairs start
  int slot;                           // of a chunk's sums; -1: the unit is the whole block
};

template <typename T>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_window_bwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_do,
                const __grid_constant__ CUtensorMap tmap_dq, T* __restrict__ dk, T* __restrict__ dv, const WindowParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  if (smem - smem_raw > kBwdSlack - kUnitBytes) {        // cannot happen while the kernel has no static shared memory
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 1);
    return;
  }
  uint8_t* sK = smem;
  uint8_t* sV = smem + kTile;
  uint8_t* sQ = smem + 2 * kTile;                    // [2][kTile]
  uint8_t* sdO = smem + 4 * kTile;
  uint8_t* sS = smem + 5 * kTile;                    // dS^T [keys x queries]
  uint8_t* sStage = smem + 6 * kTile;                // [2][kStage] fp32 dQ
  float* s_lse = reinterpret_cast<float*>(smem + 6 * kTile + 2 * kStage);   // [2][128]
  float* s_dlt = s_lse + 2 * 128;                                             // [2][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_dlt + 2 * 128);
  uint64_t* kv_full = bars;                  // 1
  uint64_t* q_full = bars + 1;               // [2]
  uint64_t* q_empty = bars + 3;              // [2]  tcgen05.commit after dK
  uint64_t* do_full = bars + 5;              // 1
  uint64_t* do_empty = bars + 6;             // tcgen05.commit after dV
  uint64_t* s_full = bars + 7;               // tcgen05.commit: S^T
  uint64_t* dp_full = bars + 8;              // tcgen05.commit: dP^T (and with it everything issued before)
  uint64_t* p_ready = bars + 9;              // 8 warps: P^T in TMEM
  uint64_t* ds_ready = bars + 10;            // 8 warps: dS^T in shared memory, dP^T read
  uint64_t* dq_full = bars + 11;             // tcgen05.commit: dQ
  uint64_t* dq_drained = bars + 12;          // 4 warps: dQ is in registers
  uint64_t* all_done = bars + 13;            // tcgen05.commit: dV, dK complete
  uint64_t* ld_full = bars + 14;             // [2]  lse and delta of a query block are there
  uint64_t* ld_empty = bars + 16;            // [2]  8 warps
  uint64_t* acc_empty = bars + 18;           // 8 warps: dV and dK of the unit are in registers
  uint64_t* u_full = bars + 19;              // [2]  a unit's description is there
  uint64_t* u_empty = bars + 21;             // [2]  all have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  BwdUnit* s_unit = reinterpret_cast<BwdUnit*>(tmem_slot + 2);     // [2]
  static_assert(23 * 8 + 8 + 2 * sizeof(BwdUnit) <= 256 + kUnitBytes, "barriers and units share this space");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_bh = p.B * p.Hkv, G = p.H / p.Hkv;
  auto complete = [&](BwdUnit& u, int chunks) {        // from kb, chunk, b and hk
    u.bh = u.b * p.Hkv + u.hk;
    u.k0 = u.kb * BK;
    // this instance's sequence (see the forward kernel): rows past a packed sequence's end are loaded, masked by index
    // (their probabilities and score gradients are exact zeros) and never stored
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
    int end;
    window_queries(p, u.kb, u.Sq, u.Sk, query_blocks(p, u.b), u.i0, end);
    u.n_i = end - u.i0;
    u.n_it = u.n_i * G;
    u.h0 = u.hk * G;
    u.slot = -1;
    if (u.kb < p.sink_blocks && chunks > 1) {         // pairs [chunk * per, (chunk + 1) * per) of this block's
      u.slot = first_slot(p, u.b) + u.chunk;
      const int per = (u.n_it + chunks - 1) / chunks, from = min(u.n_it, u.chunk * per);
      u.n_it = min(u.n_it, from + per) - from;
      if (u.n_i > 0) {
        u.h0 += from / u.n_i;
        u.istart = from % u.n_i;
      }
    }
  };
  // calls f() for every unit of this CTA until it returns false
  auto each_unit = [&](auto whole_warp, auto f) {
    for (uint32_t n = 0;; ++n) {
      if constexpr (decltype(whole_warp)::value) {
        if (!mbar_wait_warp(&u_full[n & 1], (n >> 1) & 1, abort_flag)) break;
      } else {
        if (!mbar_wait(&u_full[n & 1], (n >> 1) & 1, abort_flag)) break;
      }
      const BwdUnit u = s_unit[n & 1];
      if constexpr (decltype(whole_warp)::value) __syncwarp();
      if (!decltype(whole_warp)::value || lane == 0) mbar_arrive(&u_empty[n & 1]);
      if (u.kb < 0 || !f(u)) break;
    }
  };

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(kv_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&ld_full[i], 1);
      mbar_init(&ld_empty[i], 8);
      mbar_init(&u_full[i], 1);
      mbar_init(&u_empty[i], kUnitReaders);
    }
    mbar_init(do_full, 1);
    mbar_init(do_empty, 1);
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_ready, 8);
    mbar_init(ds_ready, 8);
    mbar_init(dq_full, 1);
    mbar_init(dq_drained, 4);
    mbar_init(all_done, 1);
    mbar_init(acc_empty, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
    prefetch_tmap(&tmap_do);
    prefetch_tmap(&tmap_dq);
  }
  if (warp == 13) {
    tmem_alloc(tmem_slot, kBwdTmemCols);
    tmem_relinquish();
  }
  auto key_blocks = [&](int b) { return min(p.kv_blocks, (max(0, p.cu_k[b + 1] - p.cu_k[b]) + BK - 1) / BK); };
  auto sink_units = [&](int b) { return min(key_blocks(b), p.sink_blocks) * chunks_of(p, query_blocks(p, b)); };
  auto other_units = [&](int b) { return max(0, key_blocks(b) - p.sink_blocks); };
  UnitWalk walk;
  if (warp == 15 && p.cu_q) walk.take(0, 0, p.B, lane, sink_units);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  constexpr uint32_t kColS = 0, kColDP = 128, kColDV = 256, kColDK = 384;

  if (warp >= 12) {
    regs_dec<kOtherRegs>();
    if (warp == 12) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        int gi = 0, live = 0;            // pairs and units with pairs so far: the phases of the barriers
        auto load_kv = [&](const BwdUnit& u) {
          mbar_expect_tx(kv_full, 2 * kTile);
          tma_load_4d(sK, &tmap_k, kv_full, 0, u.koff + u.k0, u.hk, u.bt);
          tma_load_4d(sK + kTile / 2, &tmap_k, kv_full, 64, u.koff + u.k0, u.hk, u.bt);
          tma_load_4d(sV, &tmap_v, kv_full, 0, u.koff + u.k0, u.hk, u.bt);
          tma_load_4d(sV + kTile / 2, &tmap_v, kv_full, 64, u.koff + u.k0, u.hk, u.bt);
        };
        each_unit(std::false_type{}, [&](const BwdUnit& u) -> bool {
          if (u.n_it == 0) return true;
          if (live == 0) load_kv(u);
          int h = u.h0, i = u.istart;
          for (int it = 0; it < u.n_it; ++it, ++gi) {
            const int q0 = (u.i0 + i) * BQ, st = gi & 1;
            if (!mbar_wait(&q_empty[st], (uint32_t)(((gi >> 1) & 1) ^ 1), abort_flag)) return false;
            mbar_expect_tx(&q_full[st], kTile);
            tma_load_4d(sQ + st * kTile, &tmap_q, &q_full[st], 0, u.qoff + q0, h, u.bt);
            tma_load_4d(sQ + st * kTile + kTile / 2, &tmap_q, &q_full[st], 64, u.qoff + q0, h, u.bt);
            if (!mbar_wait(do_empty, (uint32_t)((gi & 1) ^ 1), abort_flag)) return false;
            mbar_expect_tx(do_full, kTile);
            tma_load_4d(sdO, &tmap_do, do_full, 0, u.qoff + q0, h, u.bt);
            tma_load_4d(sdO + kTile / 2, &tmap_do, do_full, 64, u.qoff + q0, h, u.bt);
            if (it == 0 && live > 0) {       // K and V are free when every product of the unit before is done
              if (!mbar_wait(all_done, (uint32_t)((live - 1) & 1), abort_flag)) return false;
              load_kv(u);
            }
            if (++i == u.n_i) { i = 0; ++h; }
          }
          ++live;
          return true;
        });
      }
      __syncwarp();
    } else if (warp == 13) {
      // ------------------------------------------------------------ MMA issuer (the whole warp waits, one lane issues)
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_kk = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
      constexpr uint32_t idesc_kmn = idesc_kk | (1u << 16);                 // B read MN-major
      constexpr uint32_t idesc_mnmn = idesc_kk | (1u << 15) | (1u << 16);   // A and B read MN-major
      const bool issuer = elect_one();
      auto wait = [&](uint64_t* bar, int n) { return mbar_wait_warp(bar, (uint32_t)(n & 1), abort_flag); };
      auto kdesc = [&](const uint8_t* tile) { return make_desc(smem_u32(tile), 16, 1024); };            // read K-major
      auto mndesc = [&](const uint8_t* tile) { return make_desc(smem_u32(tile), kTile / 2, 1024); };    // read MN-major
      const uint64_t dK_k = kdesc(sK), dV_k = kdesc(sV), dO_k = kdesc(sdO), dQ_k = kdesc(sQ), dS_k = kdesc(sS);
      const uint64_t dK_mn = mndesc(sK), dO_mn = mndesc(sdO), dQ_mn = mndesc(sQ), dS_mn = mndesc(sS);
      auto koff16 = [](int kk) { return (uint32_t)(((kk >> 2) * (kTile / 2) + (kk & 3) * 32) >> 4); };   // K-major: two 64-column atoms
      auto mnoff16 = [](int kk) { return (uint32_t)((kk * 2048) >> 4); };                                // MN-major: 16 rows of 128 bytes
      int base = 0, live = 0;              // pairs before this unit's, units with pairs so far
      each_unit(std::true_type{}, [&](const BwdUnit& u) -> bool {
        if (u.n_it == 0) return true;
        bool ok = wait(kv_full, live) && wait(&q_full[base & 1], base >> 1);
        // the rows of the current and the next query block that are the sequence's own (128 or more: all)
        int mi = u.istart;
        auto own_rows = [&]() { return u.Sq - (u.i0 + mi) * BQ; };
        if (ok && p.cu_q) {
          if (u.k0 + BK > u.Sk) {
            zero_tail(sK, u.Sk - u.k0, lane);
            zero_tail(sV, u.Sk - u.k0, lane);
          }
          if (own_rows() < BQ) zero_tail(sQ + (base & 1) * kTile, own_rows(), lane);
        }
        if (ok) {
          tc_fence_after();
          if (issuer) {
            const uint32_t tq = (uint32_t)((base & 1) * (kTile >> 4));
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) umma_f16(tmem_base + kColS, dK_k + koff16(kk), dQ_k + tq + koff16(kk), idesc_kk, kk != 0 ? 1u : 0u);
            umma_commit(s_full);
          }
        }
        for (int it = 0; it < u.n_it && ok; ++it) {
          const int gi = base + it;
          const uint32_t tq = (uint32_t)((gi & 1) * (kTile >> 4)), tq_next = (uint32_t)(((gi + 1) & 1) * (kTile >> 4));
          if (!wait(do_full, gi)) { ok = false; break; }
          if (p.cu_q && own_rows() < BQ) zero_tail(sdO, own_rows(), lane);
          if (gi > 0 && !wait(dq_drained, gi - 1)) { ok = false; break; }
          tc_fence_after();
          if (issuer) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) umma_f16(tmem_base + kColDP, dV_k + koff16(kk), dO_k + koff16(kk), idesc_kk, kk != 0 ? 1u : 0u);
            umma_commit(dp_full);                        // dP^T = V dO^T
          }
          if (!wait(p_ready, gi)) { ok = false; break; }
          if (it == 0 && live > 0 && !wait(acc_empty, live - 1)) { ok = false; break; }
          tc_fence_after();
          if (issuer) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)               // dV += P^T dO; P^T of 64 queries over the left of its half of S^T
              umma_f16_ts(tmem_base + kColDV, tmem_base + kColS + (uint32_t)((kk >> 2) * 64 + (kk & 3) * 8), dO_mn + mnoff16(kk),
                          idesc_kmn, (it == 0 && kk == 0) ? 0u : 1u);
            umma_commit(do_empty);
          }
          if (it + 1 < u.n_it) {
            if (!wait(&q_full[(gi + 1) & 1], (gi + 1) >> 1)) { ok = false; break; }
            if (++mi == u.n_i) mi = 0;
            if (p.cu_q && own_rows() < BQ) zero_tail(sQ + ((gi + 1) & 1) * kTile, own_rows(), lane);
            tc_fence_after();
            if (issuer) {
#pragma unroll
              for (int kk = 0; kk < 8; ++kk)             // S^T of the next pair, over P^T of this one
                umma_f16(tmem_base + kColS, dK_k + koff16(kk), dQ_k + tq_next + koff16(kk), idesc_kk, kk != 0 ? 1u : 0u);
              umma_commit(s_full);
            }
          }
          if (!wait(ds_ready, gi)) { ok = false; break; }
          tc_fence_after();
          if (issuer) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)               // dQ = dS K over the consumed dP^T
              umma_f16(tmem_base + kColDP, dS_mn + mnoff16(kk), dK_mn + mnoff16(kk), idesc_mnmn, kk != 0 ? 1u : 0u);
            umma_commit(dq_full);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)               // dK += dS^T Q
              umma_f16(tmem_base + kColDK, dS_k + koff16(kk), dQ_mn + tq + mnoff16(kk), idesc_kmn, (it == 0 && kk == 0) ? 0u : 1u);
            umma_commit(&q_empty[gi & 1]);
            if (it + 1 == u.n_it) umma_commit(all_done);
          }
        }
        base += u.n_it;
        ++live;
        return ok;
      });
      __syncwarp();
    } else if (warp == 14) {
      // ------------------------------------------------------------ lse (log2 domain, negated: an addend of the exponent) and
      // delta (negated) of every query block; an lse of -inf switches a row off (read one block ahead, all eight loads in flight at
      // once)
      int h, i, gi = 0;
      float l[4], d[4];
      auto fetch = [&](const BwdUnit& u) {
        const int64_t base = p.cu_q ? (int64_t)h * p.total_q + u.qoff : ((int64_t)u.b * p.H + h) * p.Sq;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int qi = (u.i0 + i) * BQ + e * 32 + lane;
          l[e] = qi < u.Sq ? __ldg(p.lse + base + qi) : -INFINITY;
          d[e] = qi < u.Sq ? __ldg(p.delta + base + qi) : 0.f;
        }
      };
      each_unit(std::true_type{}, [&](const BwdUnit& u) -> bool {
        h = u.h0;
        i = u.istart;
        if (u.n_it > 0) fetch(u);
        for (int it = 0; it < u.n_it; ++it, ++gi) {
          const int st = gi & 1;
          if (!mbar_wait_warp(&ld_empty[st], (uint32_t)(((gi >> 1) & 1) ^ 1), abort_flag)) return false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s_lse[st * 128 + e * 32 + lane] = l[e] > -INFINITY ? -l[e] * 1.4426950408889634f : -INFINITY;
            s_dlt[st * 128 + e * 32 + lane] = -d[e];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&ld_full[st]);
          if (++i == u.n_i) { i = 0; ++h; }
          if (it + 1 < u.n_it) fetch(u);
        }
        return true;
      });
    } else {
      // ------------------------------------------------------------ the units, one after the other; kb < 0 behind the last
      bool in_sinks = true;
      int with_sinks = 0;
      for (uint32_t n = 0;; ++n) {
        const int unit = (int)(n * gridDim.x + (n & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x));
        BwdUnit u{};
        bool there;
        if (p.cu_q) {
          const int x = unit / p.Hkv;
          if (in_sinks && !walk.find(x, p.B, lane, u.b, u.kb, sink_units)) {
            in_sinks = false;
            with_sinks = walk.before;
            walk.take(0, 0, p.B, lane, other_units);
          }
          there = in_sinks || walk.find(x - with_sinks, p.B, lane, u.b, u.kb, other_units);
          u.hk = unit % p.Hkv;
          if (!in_sinks) u.kb += p.sink_blocks;
        } else {
          const int pairs = p.sink_blocks * chunks_of(p, p.q_blocks), bh = unit % n_bh;
          there = unit < p.units;
          u.kb = unit / n_bh;
          u.b = bh / p.Hkv;
          u.hk = bh - u.b * p.Hkv;
          in_sinks = u.kb < pairs;
          if (!in_sinks) u.kb -= pairs - p.sink_blocks;
        }
        if (there) {
          const int chunks = chunks_of(p, query_blocks(p, u.b));
          if (in_sinks) {                     // numbers of (block, chunk) pairs
            u.chunk = u.kb % chunks;
            u.kb /= chunks;
          }
          complete(u, chunks);
        } else {
          u.kb = -1;
        }
        if (!mbar_wait_warp(&u_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag)) break;
        if (lane == 0) {
          s_unit[n & 1] = u;
          mbar_arrive(&u_full[n & 1]);
        }
        __syncwarp();
        if (!there) break;
      }
    }
  } else if (warp >= 8) {
    regs_inc<kDqRegs>();
    // ------------------------------------------------------------ dQ warpgroup: TMEM -> registers -> shared memory -> global
    const int qw = warp & 3;
    const int r = qw * 32 + lane;                 // query row inside the block = TMEM lane
    const uint32_t addr = tmem_base + ((uint32_t)(qw * 32) << 16) + kColDP;
    int gi = 0;
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {        // the description stays in shared memory, as in the compute warps
      ok = mbar_wait_warp(&u_full[n & 1], (n >> 1) & 1, abort_flag);
      if (!named_bar_and(1, 128, ok)) break;                          // one answer for the four warps, here and below
      const volatile BwdUnit& u = s_unit[n & 1];
      if (u.kb < 0) break;
      const int n_it = u.n_it;
      int h = u.h0, i = u.istart;
      for (int it = 0; it < n_it && ok; ++it, ++gi) {
        const int q0 = (u.i0 + i) * BQ;
        ok = mbar_wait_warp(dq_full, (uint32_t)(gi & 1), abort_flag);
        tc_fence_after();
        uint32_t raw[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(addr + (uint32_t)(c * 32), raw[c]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dq_drained);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x0, x1;
            mul2(x0, x1, __uint_as_float(raw[c][e]), __uint_as_float(raw[c][e + 1]), p.scale, p.scale);
            raw[c][e] = __float_as_uint(x0);
            raw[c][e + 1] = __float_as_uint(x1);
          }
        if (q0 + r >= u.Sq) {        // a row of the next sequence or head: zero, also where this one's keys are not finite
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) raw[c][e] = 0u;
        }
        const int row0 = p.cu_q ? (int)((int64_t)h * p.total_q + u.qoff + q0) : (int)(((int64_t)u.b * p.H + h) * p.Sq + q0);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          // the reduction that read this box two chunks ago has finished with it
          if (threadIdx.x == 8 * 32) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          if (!named_bar_and(1, 128, ok)) { ok = false; break; }
          uint8_t* box = sStage + (c & 1) * kStage + (size_t)r * 128;
#pragma unroll
          for (int ch = 0; ch < 8; ++ch)
            *reinterpret_cast<uint4*>(box + (size_t)((ch ^ (r & 7)) * 16)) =
                make_uint4(raw[c][ch * 4], raw[c][ch * 4 + 1], raw[c][ch * 4 + 2], raw[c][ch * 4 + 3]);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          named_bar_sync(1, 128);
          if (threadIdx.x == 8 * 32) {
            tma_reduce_add_2d(&tmap_dq, sStage + (c & 1) * kStage, c * 32, row0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
        if (++i == u.n_i) { i = 0; ++h; }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&u_empty[n & 1]);
    }
    // every reduction must have completed before the CTA exits
    if (threadIdx.x == 8 * 32) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else {
    regs_inc<kComputeRegs>();
    // ------------------------------------------------------------ two compute warpgroups (warps 0-3, 4-7)
    const int wg = warp >> 2;
    const int qw = warp & 3;
    const int r = qw * 32 + lane;                 // key row inside the block = TMEM lane
    const uint32_t lane_base = ((uint32_t)(qw * 32) << 16);
    const uint32_t s_addr = tmem_base + lane_base + kColS + (uint32_t)(wg * 64);
    const uint32_t dp_addr = tmem_base + lane_base + kColDP + (uint32_t)(wg * 64);
    uint8_t* srow = sS + (size_t)wg * (kTile / 2) + (size_t)r * 128;   // this warpgroup's 64 query columns = atom `wg`
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_warp(bar, parity, abort_flag); };
    int gi = 0, live = 0;
    // The description stays in shared memory until the unit is stored: what the loop does not need would take registers from it.
    for (uint32_t n = 0;; ++n) {
      if (!wait_all(&u_full[n & 1], (n >> 1) & 1)) break;
      const volatile BwdUnit& u = s_unit[n & 1];
      const int n_it = u.n_it, i0 = u.i0, n_i = u.n_i, k0 = u.k0, Sk = u.Sk;
      if (u.kb < 0) break;
      const int kj = k0 + r;
      const bool key_off = kj >= Sk;
      const bool block_off = k0 + BK > Sk;
      const int far = kj >= p.sinks ? kj + p.window : 0x7fffffff;      // the first query that no longer sees this key
      bool ok = true;
      int i = u.istart;
      for (int it = 0; it < n_it; ++it, ++gi) {
        const uint32_t par = (uint32_t)(gi & 1);
        const int st = gi & 1, q0 = (i0 + i) * BQ;
        const float4* nlse4 = reinterpret_cast<const float4*>(s_lse + st * 128 + wg * 64);
        const float4* ndlt4 = reinterpret_cast<const float4*>(s_dlt + st * 128 + wg * 64);
        // only then can a query be older than a key of this block, a key be past the end or in front of a window
        const bool masked = q0 < k0 + BK || block_off || q0 + BQ - k0 > p.window;
        if (!wait_all(&ld_full[st], (uint32_t)((gi >> 1) & 1)) || !wait_all(s_full, par)) { ok = false; break; }
        tc_fence_after();
        float pf[64];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t raw[32], pk[16];
          tmem_ld32(s_addr + (uint32_t)(c * 32), raw);
          tmem_ld_wait();
          if (masked) {              // what is not seen becomes -inf
            const int q = q0 + wg * 64 + c * 32;
            const uint32_t seen = key_off ? 0u : low_bits(far - q) & ~low_bits(kj - q);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((seen >> e) & 1u)) raw[e] = 0xff800000u;
          }
#pragma unroll
          for (int e4 = 0; e4 < 8; ++e4) {
            const float4 nl = nlse4[c * 8 + e4];
            const float nls[4] = {nl.x, nl.y, nl.z, nl.w};
#pragma unroll
            for (int e2 = 0; e2 < 4; e2 += 2) {
              const int e = e4 * 4 + e2, cc = c * 32 + e;
              float x0, x1;
              fma2v(x0, x1, __uint_as_float(raw[e]), __uint_as_float(raw[e + 1]), p.scale_log2, nls[e2], nls[e2 + 1]);
              float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
              pf[cc] = p0;
              pf[cc + 1] = p1;
              pk[e >> 1] = pack2<T>(p0, p1);
            }
          }
          tmem_st16(s_addr + (uint32_t)(c * 16), pk);   // over columns of S^T that this thread has read
        }
        if (q0 == 0 && wg == 0) pf[0] = 0.f;      // the first query sees one key: its softmax is constant, and so dS is zero, not nearly zero
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        // dP^T; its commit also says that the products which read the previous dS^T have completed
        if (!wait_all(dp_full, par)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t raw[32], pk[16];
          tmem_ld32(dp_addr + (uint32_t)(c * 32), raw);
          tmem_ld_wait();
#pragma unroll
          for (int e4 = 0; e4 < 8; ++e4) {
            const float4 nd = ndlt4[c * 8 + e4];
            const float nds[4] = {nd.x, nd.y, nd.z, nd.w};
#pragma unroll
            for (int e2 = 0; e2 < 4; e2 += 2) {
              const int e = e4 * 4 + e2, cc = c * 32 + e;
              float t0 = __uint_as_float(raw[e]), t1 = __uint_as_float(raw[e + 1]), d0, d1;
              add2(t0, t1, nds[e2], nds[e2 + 1]);
              mul2(d0, d1, pf[cc], pf[cc + 1], t0, t1);
              pk[e >> 1] = pack2<T>(d0, d1);
            }
          }
#pragma unroll
          for (int g8 = 0; g8 < 4; ++g8) {
            const int ch = c * 4 + g8;
            *reinterpret_cast<uint4*>(srow + (size_t)((ch ^ (r & 7)) * 16)) =
                make_uint4(pk[g8 * 4], pk[g8 * 4 + 1], pk[g8 * 4 + 2], pk[g8 * 4 + 3]);
          }
        }
        tc_fence_before();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(ds_ready);
          mbar_arrive(&ld_empty[st]);
        }
        if (++i == n_i) i = 0;
      }
      if (ok && n_it > 0) ok = wait_all(all_done, (uint32_t)(live & 1));
      // ---- dK, dV of this key block
      if (ok) {
        tc_fence_after();
        const bool row_ok = kj < Sk;
        T* dk_row = dk + (int64_t)u.bt * p.dk_sb + (int64_t)u.hk * p.dk_sh + (int64_t)(u.koff + kj) * p.dk_ss + wg * 64;
        T* dv_row = dv + (int64_t)u.bt * p.dv_sb + (int64_t)u.hk * p.dv_sh + (int64_t)(u.koff + kj) * p.dv_ss + wg * 64;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t raw[32];
            if (n_it > 0) {
              tmem_ld32(tmem_base + lane_base + (which ? kColDK : kColDV) + (uint32_t)(wg * 64 + c * 32), raw);
              tmem_ld_wait();
              if (which) {
#pragma unroll
                for (int e = 0; e < 32; ++e) raw[e] = __float_as_uint(__uint_as_float(raw[e]) * p.scale);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) raw[e] = 0u;
            }
            if (u.slot >= 0) {
              float* dst = p.sink_ws + ((((int64_t)u.slot * p.sink_blocks + u.kb) * p.Hkv + u.hk) * 2 + which) * (BK * BD) + r * BD +
                           wg * 64 + c * 32;
              if (n_it > 0) {
#pragma unroll
                for (int g4 = 0; g4 < 8; ++g4)
                  *reinterpret_cast<uint4*>(dst + g4 * 4) = make_uint4(raw[g4 * 4], raw[g4 * 4 + 1], raw[g4 * 4 + 2], raw[g4 * 4 + 3]);
              }
            } else if (row_ok) {
              T* dst = (which ? dk_row : dv_row) + c * 32;
#pragma unroll
              for (int g8 = 0; g8 < 4; ++g8) {
                Vec16<T> v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v.v[e] = ToF<T>::from(__uint_as_float(raw[g8 * 8 + e]));
                st16(dst + g8 * 8, v);
              }
            }
          }
        }
      }
      if (n_it > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty);
        ++live;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&u_empty[n & 1]);
      if (!ok) break;
    }
    if (p.cu_q) {                                    // packed rows past the last sequence: zeros, the CTAs share them
      Vec16<T> zero;
#pragma unroll
      for (int e = 0; e < 8; ++e) zero.v[e] = ToF<T>::from(0.f);
      for (int64_t row = p.cu_k[p.B] + (int)blockIdx.x * 16 + (threadIdx.x >> 4); row < p.total_k; row += gridDim.x * 16)
        for (int y = 0; y < p.Hkv; ++y) {
          st16(dk + (int64_t)y * p.dk_sh + row * p.dk_ss + (threadIdx.x & 15) * 8, zero);
          st16(dv + (int64_t)y * p.dv_sh + row * p.dv_ss + (threadIdx.x & 15) * 8, zero);
        }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kBwdTmemCols);
  }
  settle_abort(abort_flag, p.status);
}

// dV and dK of the blocks with sinks of sequences that have more than one chunk: the chunks' sums, added in order (the same for every run)
// and rounded once.  Eight blocks a sequence, key block and key head; a thread owns eight dimensions of a row.  Where there are more packed
// sequences than places, the blocks go by places, and those of a sequence's first one do its work.
template <typename T>
__global__ void __launch_bounds__(256) attn_sink_sum_kernel(T* __restrict__ dk, T* __restrict__ dv, const WindowParams p) {
  const int which = blockIdx.y, r = (int)(blockIdx.x % 8) * 16 + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 8;
  const int unit = (int)(blockIdx.x / 8), kb = unit / p.Hkv, hk = unit - kb * p.Hkv, kj = kb * BK + r;
  int b = (int)blockIdx.z, Sk = p.Sk, Sq = p.Sq, koff = 0, bt = b;
  if (p.cu_q) {
    if (p.sink_slots < p.B) {            // the last sequence whose places start here or before
      int above = p.B;
      b = 0;
      while (above - b > 1) {
        const int mid = (b + above) >> 1;
        if (first_slot(p, mid) <= (int)blockIdx.z) b = mid; else above = mid;
      }
      if (first_slot(p, b) != (int)blockIdx.z) return;
    }
    koff = p.cu_k[b];
    Sk = p.cu_k[b + 1] - koff;
    Sq = p.cu_q[b + 1] - p.cu_q[b];
    bt = 0;
  }
  const int slot = first_slot(p, b);
  const int q_blocks = query_blocks(p, b), chunks = chunks_of(p, q_blocks);
  if (chunks == 1 || kj >= Sk) return;
  int first, end;
  window_queries(p, kb, Sq, Sk, q_blocks, first, end);
  const int n_it = (end - first) * (p.H / p.Hkv), per = (n_it + chunks - 1) / chunks;
  float s[8] = {};
  const float* src = p.sink_ws + ((((int64_t)slot * p.sink_blocks + kb) * p.Hkv + hk) * 2 + which) * (BK * BD) + r * BD + c;
  for (int ch = 0; ch * per < n_it; ++ch, src += (int64_t)p.sink_blocks * p.Hkv * 2 * BK * BD) {
    const float4 x = *reinterpret_cast<const float4*>(src), y = *reinterpret_cast<const float4*>(src + 4);
    s[0] += x.x; s[1] += x.y; s[2] += x.z; s[3] += x.w;
    s[4] += y.x; s[5] += y.y; s[6] += y.z; s[7] += y.w;
  }
  Vec16<T> o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o.v[e] = ToF<T>::from(s[e]);
  if (which) st16(dk + (int64_t)bt * p.dk_sb + (int64_t)hk * p.dk_sh + (int64_t)(koff + kj) * p.dk_ss + c, o);
  else st16(dv + (int64_t)bt * p.dv_sb + (int64_t)hk * p.dv_sh + (int64_t)(koff + kj) * p.dv_ss + c, o);
}

// How the query blocks of the key blocks with sinks are cut.  A chunk is about as long as what the other key blocks meet, but never so
// short that there were more than four chunks an SM: that is enough to even the units out, and it bounds the scratch by the
// machine (128 KB a chunk; at most 1776, 222 MiB) whatever the lengths and however many sinks.  Cut by the longest sequence for all, one
// sequence of 8192 tokens and 199 of under 60 (8 key heads, window 128, four sinks) took 6.4 GB and 1340 us, now 0.1 GB and 620; 16384
// tokens with 4 heads, window 128 and 4096 sinks 1.0 GB and 970 us, now 0.1 GB and 440; 32 heads x 4096, window 64, four sinks 257 us,
// now 241.
struct SinkPlan {
  int blocks, chunk, slots;
};
SinkPlan sink_plan(const b200_attn_t* a) {
  SinkPlan s{0, 1, 0};
  if (a->window <= 0 || a->sinks <= 0 || a->B <= 0 || a->Hkv <= 0 || a->Sq <= 0 || a->Sk <= 0) return s;
  const bool packed = a->cu_seqlens_q != nullptr;
  const long long q_blocks = (a->Sq + BQ - 1) / BQ, all = packed ? ((long long)a->total_q + BQ - 1) / BQ : a->B * q_blocks;
  s.blocks = (std::min(a->sinks, a->Sk) + BK - 1) / BK;
  const long long others = (a->window + BK - 2ll) / BQ + 1, even = (all * a->Hkv * s.blocks + 4 * kSMs - 1) / (4 * kSMs);
  s.chunk = (int)std::min(q_blocks, std::max(others, even));
  if (q_blocks > s.chunk) s.slots = packed ? slots_before(a->total_q, s.chunk) : (int)(a->B * ((q_blocks + s.chunk - 1) / s.chunk));
  return s;
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int64_t b200_flash_attn_bwd_workspace(const b200_attn_t* a) {
  const SinkPlan s = sink_plan(a);
  return (int64_t)s.slots * s.blocks * a->Hkv * 2 * BK * BD;
}

namespace b200k {

int attn_window_bwd(const b200_attn_t* a, float* dq_accum, void* dk, void* dv, float* delta, const void* q, const void* k, const void* v,
                    const void* o, const void* d_o, const float* lse, const int64_t* extra_strides, cudaStream_t stream) {
  BwdMaps m;
  if (int e = bwd_maps(&m, a, dq_accum, dk, dv, q, k, v, o, d_o, extra_strides)) return e;
  const int64_t* x = extra_strides;
  WindowParams p{};
  p.B = a->B; p.H = a->H; p.Hkv = a->Hkv; p.Sq = a->Sq; p.Sk = a->Sk;
  p.scale = a->window == 1 && a->sinks == 0 ? 0.f : a->scale;      // every query sees one key: dS is zero
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.lse = lse;
  p.delta = delta;
  p.dq = dq_accum;
  p.dk_sb = x[3]; p.dk_sh = x[4]; p.dk_ss = x[5];
  p.dv_sb = x[6]; p.dv_sh = x[7]; p.dv_ss = x[8];
  p.kv_blocks = (a->Sk + BK - 1) / BK;
  p.q_blocks = (a->Sq + BQ - 1) / BQ;
  p.status = gemm_status_word_device();
  p.cu_q = a->cu_seqlens_q;
  p.cu_k = a->cu_seqlens_k;
  p.total_q = a->total_q;
  p.window = a->window;
  p.sinks = a->sinks;
  p.total_k = a->total_k;
  const SinkPlan plan = sink_plan(a);
  p.sink_blocks = plan.blocks;
  p.sink_chunk = plan.chunk;
  p.sink_slots = plan.slots;
  p.sink_ws = a->workspace;
  if (!a->causal || a->window > (1 << 30) || a->sinks < 0 || (plan.slots > 0 && !p.sink_ws) ||
      (reinterpret_cast<uintptr_t>(a->remainder) & 15))
    return (int)cudaErrorNotSupported;
  // of packed sequences the most there can be: only the grid follows from it, the units that exist are counted on the device
  const long long units = (long long)a->Hkv * ((long long)a->B * p.kv_blocks + (long long)plan.slots * plan.blocks -
                                               (p.cu_q || plan.slots == 0 ? 0ll : (long long)a->B * plan.blocks));
  if (units > 2147483647ll - 1024) return (int)cudaErrorNotSupported;
  p.units = (int)units;
  const unsigned grid = (unsigned)std::min<long long>(units, gemm_sm_count());
  auto launch = [&](auto kern, OncePerDevice& once, auto* gk, auto* gv) -> int {
    using T = std::remove_pointer_t<decltype(gk)>;
    if (int e = once([&] { return bwd_setup(kern); })) return e;
    auto delta_kern = a->remainder ? attn_delta_kernel<T, true> : attn_delta_kernel<T, false>;
    delta_kern<<<m.delta_grid, 256, 0, stream>>>((const T*)o, (const T*)d_o, delta, dq_accum, a->H, m.delta_rows, (int)m.row_blocks, a->o_sb,
                                                 a->o_sh, a->o_ss, x[0], x[1], x[2], (const T*)a->remainder);
    kern<<<grid, kBwdThreads, kBwdSmem, stream>>>(m.q, m.k, m.v, m.d_o, m.dq, gk, gv, p);
    note_launch(2);
    if (plan.slots > 0) {
      const unsigned z = (unsigned)std::min(plan.slots, a->B);
      attn_sink_sum_kernel<T><<<dim3((unsigned)(plan.blocks * a->Hkv * 8), 2, z), 256, 0, stream>>>(gk, gv, p);
      note_launch();
    }
    return (int)cudaGetLastError();
  };
  static OncePerDevice once[2];
  return a->dtype == B200_BF16 ? launch(attn_window_bwd_kernel<__nv_bfloat16>, once[0], (__nv_bfloat16*)dk, (__nv_bfloat16*)dv)
                               : launch(attn_window_bwd_kernel<__half>, once[1], (__half*)dk, (__half*)dv);
}

}  // namespace b200k
