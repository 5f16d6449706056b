// One pass over the new tokens of a decode or prompt step: RMSNorm of every query / key head (optional), rotary position
// embedding, and the append of keys and values to a paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                     (optional, per head of D values)
//   (a, b) <- (a cos - b sin, a sin + b cos),  angle = pos * inv_freq[i]
//
// pairs (2i, 2i + 1) or (i, i + rot / 2) of the first `rot` values; the others pass through.  The angle of a far position
// loses its digits in 32 bits (2^17 * 2^-24 is already 0.008), so it is formed and reduced to one turn in 64 bits; the
// rest is 32-bit arithmetic with one rounding to the 16-bit type at the store.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../api.h"
#include "../common/launch.h"
#include "../common/ptx.cuh"

namespace rt {

namespace {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16(v); }

// cos and sin of pos * inv_freq: product and reduction to [-pi, pi] in 64 bits, the functions in 32.
__device__ __forceinline__ void rotation(int pos, float inv_freq, float* cs, float* sn) {
  const double turns = (double)pos * (double)inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  sincosf((float)((turns - rint(turns)) * 6.283185307179586477), sn, cs);
}

// One warp per (token, head row): q heads, then k heads, then v heads.
template <typename T>
__global__ void paged_append_kernel(PagedAppendArgs a, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int rows = a.H + 2 * a.cache.Hkv;
  const long long r = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (r >= (long long)a.n_tok * rows) return;
  const int t = (int)(r / rows), h = (int)(r % rows);
  const int D = a.cache.D, half = a.rot >> 1;
  const int kind = h < a.H ? 0 : h < a.H + a.cache.Hkv ? 1 : 2;
  const int hh = kind == 0 ? h : kind == 1 ? h - a.H : h - a.H - a.cache.Hkv;
  const int p = a.pos[t], s = a.seq ? a.seq[t] : t;
  long long slot = -1;
  if (s != -1) {
    const long long pg = p / a.cache.page;
    bool ok = p >= 0 && s >= 0 && s < a.cache.n_seq && pg < a.cache.max_pages;
    if (ok) {
      const int page = a.cache.table[s * a.cache.table_stride + pg];
      ok = page >= 0 && page < a.cache.n_pages;
      slot = page * a.cache.s_page + (p % a.cache.page) * a.cache.s_row + hh * a.cache.s_head;
    }
    if (!ok) {
      slot = -1;
      if (lane == 0) atomicCAS(status, 0, RT_ERR_BOUNDS);
    }
  }
  const T* src = kind == 0 ? (const T*)a.q + t * a.q_st + hh * a.q_sh
                           : kind == 1 ? (const T*)a.k + t * a.k_st + hh * a.k_sh : (const T*)a.v + t * a.v_st + hh * a.v_sh;
  T* out = kind == 0 ? (T*)a.q_out + t * a.qo_st + hh * a.qo_sh
                     : kind == 1 && a.k_out ? (T*)a.k_out + t * a.ko_st + hh * a.ko_sh : nullptr;
  T* dst = kind == 0 || slot < 0 ? nullptr : (T*)(kind == 1 ? a.cache.k : a.cache.v) + slot;
  if (slot < 0) {  // padded or refused token: nothing is appended, its outputs are zero
    if (out)
      for (int d = lane; d < D; d += 32) out[d] = from_f<T>(0.f);
    return;
  }
  if (kind == 2) {
    for (int d = lane; d < D; d += 32) dst[d] = src[d];
    return;
  }
  const T* w = (const T*)(kind == 0 ? a.q_norm : a.k_norm);
  float r_inv = 1.f;
  if (w) {
    float ss = 0.f;
    for (int d = lane; d < D; d += 32) {
      const float x = to_f(src[d]);
      ss = fmaf(x, x, ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    r_inv = rsqrtf(ss / D + a.eps);
  }
  auto load = [&](int d) { return w ? to_f(src[d]) * r_inv * to_f(w[d]) : to_f(src[d]); };
  auto store = [&](int d, float v) {
    const T x = from_f<T>(v);
    if (out) out[d] = x;
    if (dst) dst[d] = x;
  };
  for (int i = lane; i < half; i += 32) {
    float cs, sn;
    rotation(p, a.inv_freq[i], &cs, &sn);
    const int ia = a.interleaved ? 2 * i : i, ib = a.interleaved ? 2 * i + 1 : i + half;
    const float x = load(ia), y = load(ib);
    store(ia, x * cs - y * sn);
    store(ib, x * sn + y * cs);
  }
  for (int d = a.rot + lane; d < D; d += 32) store(d, load(d));
}

}  // namespace

void paged_append(const PagedAppendArgs& a, cudaStream_t s) {
  if (a.n_tok == 0) return;
  const long long rows = (long long)a.n_tok * (a.H + 2 * a.cache.Hkv);
  const dim3 grid((unsigned)((rows + 7) / 8)), block(256);
  int* status = status_word(current_device());
  if (a.dtype == DT_F16) launch_pdl(paged_append_kernel<__half>, grid, block, 0, s, a, status);
  else launch_pdl(paged_append_kernel<__nv_bfloat16>, grid, block, 0, s, a, status);
  RT_LAUNCH_CHECK();
}

}  // namespace rt
