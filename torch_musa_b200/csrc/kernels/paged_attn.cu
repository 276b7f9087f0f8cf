// Attention of the newest tokens of each sequence over a paged key-value cache, and the rotary embedding that writes it.
//
// The cache is a pool of pages [num_pages, Hkv, page_size, D] for keys and one for values; row b of the block table names
// the pages of sequence b in order.  seq_lens[b] counts the tokens of the sequence that are in the cache, the newest
// included, so token i of n new ones stands at position len - n + i.  Everything that changes from step to step is read
// on the device, so that a captured step can be replayed.
// Parity: the reference has no paged cache; its decoding goes through the vendor SDPA on contiguous keys (reference
// torch_musa/csrc/aten/ops/attention/mudnn/SDP.cpp).
#include "common.cuh"

#include <initializer_list>

namespace b200k {
namespace {

struct PagedParams {
  int B, n, H, Hkv;
  int num_pages, page_size, table_width;
  int window, sinks;          // window <= 0: every earlier key is visible
  float scale_log2;
  int64_t q_sb, q_sn, q_sh;                    // element strides; rows of D contiguous elements
  int64_t k_sp, k_sh, k_sr, v_sp, v_sh, v_sr;  // page, head, row in the page
  int64_t table_sb;
  const int* table;
  const int* lens;
  int* status;
};

// The number of the page that holds key j of a sequence, or -1 (and a note for the host) when the table has none.
__device__ __forceinline__ int page_of(const PagedParams& p, const int* row, int index) {
  int page = -1;
  if (index < p.table_width) page = __ldg(row + index);
  if (page < 0 || page >= p.num_pages) {
    if (p.status) atomicExch(p.status, 1);
    page = -1;
  }
  return page;
}

// One warp per (sequence, new token, query head); its lanes split the D dimensions.  Online softmax in the log2 domain:
// m' = max(m, s), l' = l 2^(m - m') + 2^(s - m'), o' = o 2^(m - m') + 2^(s - m') v.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_attn_kernel(T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ kp,
                                                         const T* __restrict__ vp, const PagedParams p) {
  constexpr int E = D / 32;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (long long)p.B * p.n * p.H) return;
  const int lane = threadIdx.x & 31;
  const int h = (int)(w % p.H), i = (int)(w / p.H % p.n), b = (int)(w / p.H / p.n);
  const int hk = h / (p.H / p.Hkv);
  const long long cap = (long long)p.table_width * p.page_size;
  const int len = (int)min((long long)max(p.lens[b], 0), cap);
  const int pos = len - p.n + i;
  const int* row = p.table + b * p.table_sb;
  float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = ToF<T>::to(q[b * p.q_sb + i * p.q_sn + h * p.q_sh + lane * E + e]) * p.scale_log2;
    o[e] = 0.f;
  }
  const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  int page = -1, at = -1;
  for (int j = (p.window > 0 && p.sinks > 0) ? 0 : lo; j <= pos; ++j) {
    if (j >= p.sinks && j < lo) j = lo;
    if (j / p.page_size != at) {
      at = j / p.page_size;
      page = page_of(p, row, at);
    }
    if (page < 0) continue;
    const int64_t r = j % p.page_size;
    const T* kr = kp + page * p.k_sp + hk * p.k_sh + r * p.k_sr + lane * E;
    const T* vr = vp + page * p.v_sp + hk * p.v_sh + r * p.v_sr + lane * E;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qv[e], ToF<T>::to(kr[e]), s);
    s = warp_sum(s);
    const float m_new = fmaxf(m, s);
    const float a = m == -INFINITY ? 0.f : exp2f(m - m_new), x = s == -INFINITY ? 0.f : exp2f(s - m_new);   // a NaN score stays one
    l = l * a + x;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(x, ToF<T>::to(vr[e]), o[e] * a);
    m = m_new;
  }
  T* dst = out + w * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = ToF<T>::from(l == 0.f ? 0.f : o[e] / l);
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

template <typename T, int D>
int launch_paged(const b200_paged_attn_t* a, void* out, const void* q, const void* kp, const void* vp, const PagedParams& p,
                 cudaStream_t stream) {
  const long long warps = (long long)p.B * p.n * p.H, grid = (warps + 3) / 4;
  if (grid > 2147483647ll) return (int)cudaErrorNotSupported;
  paged_attn_kernel<T, D><<<(unsigned)grid, 128, 0, stream>>>((T*)out, (const T*)q, (const T*)kp, (const T*)vp, p);
  B200K_LAUNCH_RET();
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
  const bool bf16 = a->dtype == B200_BF16, wide = a->head_dim == 128;
  if (bf16) return wide ? launch_paged<__nv_bfloat16, 128>(a, out, q, k_pages, v_pages, p, stream)
                        : launch_paged<__nv_bfloat16, 64>(a, out, q, k_pages, v_pages, p, stream);
  return wide ? launch_paged<__half, 128>(a, out, q, k_pages, v_pages, p, stream)
              : launch_paged<__half, 64>(a, out, q, k_pages, v_pages, p, stream);
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
