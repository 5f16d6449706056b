// Attention of new tokens over a paged key / value cache:
//
//   s_j = f(scale q . K_j),  f(x) = x  or  softcap tanh(x / softcap)
//   out = sum_j exp(s_j - m) V_j / sum_j exp(s_j - m),  j in [max(0, kv_len - window), kv_len),  m = max s_j
//
// A token that sees no position gets zeros.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "../api.h"
#include "../common/launch.h"
#include "../common/ptx.cuh"

namespace rt {

namespace {

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

constexpr int PA_WARPS = 8;

// One CTA per (token, query head); each warp walks every 8th key with a running maximum, sum and output.
template <typename T>
__global__ void paged_attention_kernel(PagedAttnArgs a, int* status) {
  __shared__ float sm_acc[PA_WARPS][256];
  __shared__ float sm_m[PA_WARPS], sm_l[PA_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedCache& c = a.cache;
  const int hk = h / (a.H / c.Hkv), D = c.D;
  const int s = a.seq ? a.seq[t] : t;
  long long len = a.kv_len[t];
  if (s == -1) len = 0;
  else if (s < 0 || s >= c.n_seq || len < 0 || len > (long long)c.max_pages * c.page) {
    if (threadIdx.x == 0) atomicCAS(status, 0, RT_ERR_BOUNDS);
    len = 0;
  }
  const long long lo = a.window > 0 && len > a.window ? len - a.window : 0;
  float q[8], acc[8], m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = lane + 32 * e;
    q[e] = d < D ? to_f(((const T*)a.q)[t * a.q_st + h * a.q_sh + d]) : 0.f;
    acc[e] = 0.f;
  }
  for (long long j = lo + warp; j < len; j += PA_WARPS) {
    const int page = c.table[s * c.table_stride + j / c.page];
    if (page < 0 || page >= c.n_pages) {
      if (lane == 0) atomicCAS(status, 0, RT_ERR_BOUNDS);
      continue;
    }
    const long long off = page * c.s_page + hk * c.s_head + (j % c.page) * c.s_row;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < D) dot = fmaf(q[e], to_f(((const T*)c.k)[off + lane + 32 * e]), dot);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    dot *= a.scale;
    if (a.softcap > 0.f) dot = a.softcap * tanhf(dot / a.softcap);
    const float mn = fmaxf(m, dot), corr = expf(m - mn), p = expf(dot - mn);
    l = l * corr + p;
    m = mn;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < D) acc[e] = acc[e] * corr + p * to_f(((const T*)c.v)[off + lane + 32 * e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sm_acc[warp][lane + 32 * e] = acc[e];
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
  __syncthreads();
  float mm = -CUDART_INF_F;
  for (int w = 0; w < PA_WARPS; ++w) mm = fmaxf(mm, sm_m[w]);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float x = 0.f, ll = 0.f;
    for (int w = 0; w < PA_WARPS; ++w)
      if (sm_m[w] != -CUDART_INF_F) {
        const float f = expf(sm_m[w] - mm);
        x += f * sm_acc[w][d];
        ll += f * sm_l[w];
      }
    put((T*)a.out + t * a.o_st + h * a.o_sh + d, ll == 0.f ? 0.f : x / ll);
  }
}

}  // namespace

void paged_attention(const PagedAttnArgs& a, cudaStream_t s) {
  if (a.n_tok == 0) return;
  const dim3 grid(a.n_tok, a.H), block(PA_WARPS * 32);
  int* status = status_word(current_device());
  if (a.dtype == DT_F16) launch_pdl(paged_attention_kernel<__half>, grid, block, 0, s, a, status);
  else launch_pdl(paged_attention_kernel<__nv_bfloat16>, grid, block, 0, s, a, status);
  RT_LAUNCH_CHECK();
}

}  // namespace rt
