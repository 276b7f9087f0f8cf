// Shared by the two attention backward kernels (dense / causal, and windowed): tile sizes, the TMA reduction, the row dots, and what
// the launchers check and describe.
#pragma once

#include "attention_common.cuh"

#include <type_traits>

namespace b200k {
namespace {
using namespace gemmdev;
using namespace attndev;

constexpr int BQ = 128, BK = 128, BD = 128;
constexpr int kTile = 128 * 128 * 2;
constexpr int kStage = 128 * 32 * 4;                  // 16 KB: 32 fp32 columns of dQ
constexpr int kBwdSlack = 768;                        // for the alignment of the tiles to 1024 bytes (checked by the kernel)
constexpr int kBwdSmem = 2 * kTile /*K, V*/ + 2 * kTile /*Q*/ + kTile /*dO*/ + kTile /*dS^T*/ + 2 * kStage /*dQ*/ +
                         2 * 2 * 128 * 4 /*lse, delta*/ + 256 /*barriers*/ + kBwdSlack;
static_assert(kBwdSmem <= 232448, "exceeds the 227 KB of shared memory a CTA can have");
constexpr int kBwdThreads = 512;                      // 2 compute warpgroups, dQ warpgroup, TMA / MMA / lse-delta warps
constexpr int kComputeRegs = 136, kDqRegs = 144, kOtherRegs = 96;    // register split (sum: what 128 per thread brings)
constexpr int kLaunchRegs = (2 * kComputeRegs + kDqRegs + kOtherRegs + 3) / 4;
constexpr uint32_t kBwdTmemCols = 512;

// adds a [128 rows x 32 floats] box of shared memory (128B-swizzled) into global memory at (x, y) of the tensor map
__device__ __forceinline__ void tma_reduce_add_2d(const CUtensorMap* map, const void* smem_src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(smem_u32(smem_src)), "r"(x), "r"(y)
               : "memory");
}

inline bool make_dq_map(CUtensorMap* out, float* ptr, int64_t rows) {
  static EncodeTiledFn enc = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      return (EncodeTiledFn) nullptr;
    }
    return (EncodeTiledFn)p;
  }();
  if (!enc || rows <= 0) return false;
  cuuint64_t dims[2] = {128, (cuuint64_t)rows};
  cuuint64_t strides[1] = {128 * sizeof(float)};
  cuuint32_t box[2] = {32, 128};
  cuuint32_t estr[2] = {1, 1};
  return enc(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// delta[b, h, q] = sum_d O[b, h, q, d] * dO[b, h, q, d], and the row of the fp32 dQ buffer is zeroed on the way.  Sixteen
// lanes per row with 16-byte accesses, 64 consecutive rows of one (batch, head) per block, four rows in flight per lane:
// bound by memory (2 x 256 bytes in, 512 out per row).  32 x 4096 rows: 24 us, against 30 (8-byte loads, a row per warp,
// 64-bit divisions for its place) + 11 for the memset it replaces.  kRest: O comes with what rounding left of it.
constexpr int kDeltaRows = 64;
template <typename T, bool kRest = false>
__global__ void __launch_bounds__(256) attn_delta_kernel(const T* __restrict__ o, const T* __restrict__ d_o, float* __restrict__ delta,
                                                         float* __restrict__ dq, int H, int Sq, int row_blocks, int64_t o_sb,
                                                         int64_t o_sh, int64_t o_ss, int64_t g_sb, int64_t g_sh, int64_t g_ss,
                                                         const T* __restrict__ rest = nullptr) {
  const int bh = (int)(blockIdx.x / row_blocks);
  const int b = bh / H, h = bh - b * H;
  const int q0 = (int)(blockIdx.x - (unsigned)bh * row_blocks) * kDeltaRows + (threadIdx.x >> 4);
  const int l16 = threadIdx.x & 15;
  const T* po = o + b * o_sb + h * o_sh + l16 * 8;
  const T* pg = d_o + b * g_sb + h * g_sh + l16 * 8;
  const T* pr = rest + b * o_sb + h * o_sh + l16 * 8;
  Vec16<T> av[4], gv[4], rv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = q0 + i * 16;
    if (q < Sq) {
      av[i] = ld16(po + q * o_ss);
      gv[i] = ld16(pg + q * g_ss);
      if constexpr (kRest) rv[i] = ld16(pr + q * o_ss);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int q = q0 + i * 16;
    float s = 0.f;
    if (q < Sq) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (kRest ? ToF<T>::to(av[i].v[e]) + ToF<T>::to(rv[i].v[e]) : ToF<T>::to(av[i].v[e])) * ToF<T>::to(gv[i].v[e]);
    }
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    if (q < Sq) {
      const int64_t row = (int64_t)bh * Sq + q;
      if (l16 == 0) delta[row] = s;
      float4* z = reinterpret_cast<float4*>(dq + row * BD);
      z[l16] = make_float4(0.f, 0.f, 0.f, 0.f);
      z[l16 + 16] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
}

template <typename K>
int bwd_setup(K kern) {
  cudaFuncAttributes at;
  cudaError_t e = cudaFuncGetAttributes(&at, kern);
  if (e != cudaSuccess) return (int)e;
  if (at.numRegs < kLaunchRegs) return (int)cudaErrorNotSupported;   // the register split would wait for ever
  return opt_in_smem(kern, kBwdSmem);
}

struct BwdMaps {
  CUtensorMap q, k, v, d_o, dq;
  int delta_rows;                      // the row-dot kernel's view of o and d_o
  unsigned row_blocks, delta_grid;
};
// Checks what both kernels ask of their operands and encodes the tensor maps.
inline int bwd_maps(BwdMaps* m, const b200_attn_t* a, float* dq_accum, const void* dk, const void* dv, const void* q, const void* k, const void* v,
                    const void* o, const void* d_o, const int64_t* extra_strides) {
  // extra_strides: do_sb, do_sh, do_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss (elements)
  if (a->head_dim != BD || (a->dtype != B200_BF16 && a->dtype != B200_F16) || a->B <= 0 || a->H <= 0 || a->Hkv <= 0 ||
      a->H % a->Hkv != 0 || a->Sq <= 0 || a->Sk <= 0)
    return (int)cudaErrorNotSupported;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const int64_t* x = extra_strides;
  const int64_t strides[] = {a->q_sb, a->q_sh, a->q_ss, a->k_sb, a->k_sh, a->k_ss, a->v_sb, a->v_sh, a->v_ss,
                             a->o_sb, a->o_sh, a->o_ss, x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], x[8]};
  for (int64_t s : strides)
    if (s % 8 != 0) return (int)cudaErrorNotSupported;
  if (!al(q) || !al(k) || !al(v) || !al(o) || !al(d_o) || !al(dk) || !al(dv) || !al(dq_accum)) return (int)cudaErrorNotSupported;
  const bool packed = a->cu_seqlens_q != nullptr;
  if (packed && (!a->cu_seqlens_k || a->total_q <= 0 || a->total_k <= 0)) return (int)cudaErrorNotSupported;
  if ((a->B > 1 && !packed && (a->q_sb == 0 || a->k_sb == 0 || a->v_sb == 0 || x[0] == 0)) ||
      (a->H > 1 && (a->q_sh == 0 || x[1] == 0)) || (a->Hkv > 1 && (a->k_sh == 0 || a->v_sh == 0)) || a->q_ss == 0 ||
      a->k_ss == 0 || a->v_ss == 0 || x[2] == 0)
    return (int)cudaErrorNotSupported;
  const int bf16 = a->dtype == B200_BF16;
  CUtensorMap mq, mk, mv, mdo;
  auto nz = [](int64_t s, int64_t fallback) { return s ? s : fallback; };
  if (packed) {
    // one "batch" of total rows: the kernel adds each sequence's first row to its tile coordinates
    if (!make_attn_map(&mq, q, bf16, 1, a->H, a->total_q, (int64_t)a->total_q * a->q_ss, nz(a->q_sh, 8), a->q_ss) ||
        !make_attn_map(&mk, k, bf16, 1, a->Hkv, a->total_k, (int64_t)a->total_k * a->k_ss, nz(a->k_sh, 8), a->k_ss) ||
        !make_attn_map(&mv, v, bf16, 1, a->Hkv, a->total_k, (int64_t)a->total_k * a->v_ss, nz(a->v_sh, 8), a->v_ss) ||
        !make_attn_map(&mdo, d_o, bf16, 1, a->H, a->total_q, (int64_t)a->total_q * x[2], nz(x[1], 8), x[2]))
      return (int)cudaErrorNotSupported;
  } else if (!make_attn_map(&mq, q, bf16, a->B, a->H, a->Sq, nz(a->q_sb, 8), nz(a->q_sh, 8), a->q_ss) ||
             !make_attn_map(&mk, k, bf16, a->B, a->Hkv, a->Sk, nz(a->k_sb, 8), nz(a->k_sh, 8), a->k_ss) ||
             !make_attn_map(&mv, v, bf16, a->B, a->Hkv, a->Sk, nz(a->v_sb, 8), nz(a->v_sh, 8), a->v_ss) ||
             !make_attn_map(&mdo, d_o, bf16, a->B, a->H, a->Sq, nz(x[0], 8), nz(x[1], 8), x[2]))
    return (int)cudaErrorNotSupported;
  // dq_accum as a [B * H * Sq, 128] ([H * total_q, 128] when packed) fp32 matrix; one box = 32 columns of 128 rows
  const long long rows = packed ? (long long)a->H * a->total_q : (long long)a->B * a->H * a->Sq;
  const int dB = packed ? 1 : a->B, dS = packed ? a->total_q : a->Sq;     // the row-dot kernel's view of o and d_o
  CUtensorMap mdq;
  if (!make_dq_map(&mdq, dq_accum, rows)) return (int)cudaErrorNotSupported;
  m->q = mq; m->k = mk; m->v = mv; m->d_o = mdo; m->dq = mdq;
  m->delta_rows = dS;
  m->row_blocks = (unsigned)((dS + kDeltaRows - 1) / kDeltaRows);
  if (rows / 8 + 1 > 2147483647ll) return (int)cudaErrorNotSupported;
  m->delta_grid = (unsigned)((long long)dB * a->H * m->row_blocks);
  return 0;
}

}  // namespace

// the windowed backward (attention_window_bwd.cu), which b200_flash_attn_bwd hands its calls with a window to
int attn_window_bwd(const b200_attn_t* a, float* dq_accum, void* dk, void* dv, float* delta, const void* q, const void* k, const void* v,
                    const void* o, const void* d_o, const float* lse, const int64_t* extra_strides, cudaStream_t stream);
}  // namespace b200k
