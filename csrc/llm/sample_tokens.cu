// Drawing one token a row from given random numbers:
//
//   w_i = exp((l_i - max l) / T)                 T = 0: the most likely token
//   order: larger l first, equal l by index;  top_k: the first k of it;  top_p: of those the shortest prefix whose mass
//   reaches top_p of theirs;  min_p: w_i >= min_p
//   token = first index (in vocabulary order) at which the running sum of the kept w exceeds u times their sum
//
// Weights are fixed-point numbers, w = round(2^45 exp(..)), so every sum of them is exact: the token does not depend on
// the order in which threads add, and a value next to a border falls on the side the 64-bit formula puts it on.  The sum
// of 2^18 weights stays below 2^63, the resolution is 3e-14 of the most likely token.  All filters keep a prefix of one
// order, so the kept set is the largest threshold of the three: keys above it, and the first few that equal it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "../api.h"
#include "../common/launch.h"
#include "../common/ptx.cuh"

namespace rt {

namespace {

typedef unsigned long long u64;
constexpr int ST_THREADS = 1024;
constexpr double ST_ONE = 35184372088832.0;  // 2^45

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// NaN counts as minus infinity, -0 as 0: equal values get equal keys.
__device__ __forceinline__ float clean(float l) { return l == l ? l + 0.f : -CUDART_INF_F; }
__device__ __forceinline__ unsigned key_of(float l) {
  const unsigned b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ u64 weight(float l, float m, double c) {
  if (l == m) return (u64)ST_ONE;
  if (l == -CUDART_INF_F) return 0;
  const double y = ((double)l - (double)m) * c;
  return y > -46.0 ? (u64)__double2ll_rn(exp2(y) * ST_ONE) : 0;
}

template <typename V, typename Op>
__device__ V block_reduce(V v, V* buf, Op op) {  // every thread gets the result
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  V r = buf[0];
  for (int w = 1; w < ST_THREADS / 32; ++w) r = op(r, buf[w]);
  return r;
}

template <typename T>
__global__ void __launch_bounds__(ST_THREADS) sample_tokens_kernel(SampleArgs a) {
  __shared__ u64 buf[ST_THREADS / 32];
  __shared__ u64 pre[ST_THREADS];
  __shared__ int pre_n[ST_THREADS];
  __shared__ int sm_pick;
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, V = a.vocab, tid = threadIdx.x;
  const T* x = (const T*)a.logits + row * a.ld;
  auto at = [&](int i) { return clean(to_f(x[i])); };
  auto add = [](u64 p, u64 q) { return p + q; };

  // most likely token: largest key, lowest index
  u64 best = 0;
  for (int i = tid; i < V; i += ST_THREADS) {
    const u64 k = ((u64)key_of(at(i)) << 32) | (unsigned)~i;
    best = k > best ? k : best;
  }
  best = block_reduce(best, buf, [](u64 p, u64 q) { return p > q ? p : q; });
  const float m = of_key((unsigned)(best >> 32));
  const double T_ = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
  if (m == -CUDART_INF_F || !(T_ > 0.0)) {
    if (tid == 0) a.out[row] = m == -CUDART_INF_F ? -1 : (long long)(int)~(unsigned)best;
    return;
  }
  const double c = 1.4426950408889634074 / T_;
  const int top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
  const double top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
  const double min_w = (a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p) * ST_ONE;

  // sum of f(key) over keys >= t
  auto above = [&](unsigned t, bool mass) {
    u64 v = 0;
    for (int i = tid; i < V; i += ST_THREADS) {
      const float l = at(i);
      if (key_of(l) >= t) v += mass ? weight(l, m, c) : 1;
    }
    return block_reduce(v, buf, add);
  };
  // largest key t with above(t) >= want (the lowest key of all when there is none)
  auto search = [&](u64 want, bool mass) {
    unsigned t = 0;
    for (int b = 31; b >= 0; --b)
      if (above(t | (1u << b), mass) >= want) t |= 1u << b;
    return t;
  };
  unsigned cut = 0;       // kept: keys > cut, and the first `ties` that equal it
  u64 ties = (u64)V;
  u64 total;
  if (top_k > 0 && top_k < V) {
    cut = search((u64)top_k, false);
    const u64 over = cut == 0xffffffffu ? 0 : above(cut + 1, false);
    ties = (u64)top_k - over;
    total = (cut == 0xffffffffu ? 0 : above(cut + 1, true)) + ties * weight(of_key(cut), m, c);
  } else {
    total = above(0, true);
  }
  if (top_p < 1.0) {
    const double want = ceil((top_p > 0.0 ? top_p : 0.0) * (double)total);
    const u64 thr = want >= 1.0 ? (want < (double)total ? (u64)want : total) : 1;
    const unsigned t = search(thr, true);
    if (t >= cut) {
      const u64 over = t == 0xffffffffu ? 0 : above(t + 1, true), w = weight(of_key(t), m, c);
      const u64 n = w ? (thr - over + w - 1) / w : 1;
      ties = t == cut && n > ties ? ties : n;
      cut = t;
    }
  }

  // draw: contiguous stretches per thread, ties counted along the index
  const int per = (V + ST_THREADS - 1) / ST_THREADS, i0 = min(V, tid * per), i1 = min(V, i0 + per);
  int n_eq = 0;
  for (int i = i0; i < i1; ++i) n_eq += key_of(at(i)) == cut;
  pre_n[tid] = n_eq;
  __syncthreads();
  u64 eq = 0;
  for (int w = 0; w < tid; ++w) eq += pre_n[w];
  auto kept = [&](int i, u64& eq_before) -> u64 {
    const float l = at(i);
    const unsigned k = key_of(l);
    const bool in = k > cut || (k == cut && eq_before < ties);
    eq_before += k == cut;
    const u64 w = in ? weight(l, m, c) : 0;
    return l == m || (double)w >= min_w ? w : 0;
  };
  u64 mass = 0, e = eq;
  for (int i = i0; i < i1; ++i) mass += kept(i, e);
  pre[tid] = mass;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int w = 0; w < ST_THREADS; ++w) {
    if (w < tid) before += pre[w];
    all += pre[w];
  }
  double u = a.uniform_f64 ? ((const double*)a.uniform)[row] : (double)((const float*)a.uniform)[row];
  u = u > 0.0 ? u : 0.0;
  const u64 target = __umul64hi(u < 1.0 ? (u64)(u * 18446744073709551616.0) : ~0ull, all);
  if (target >= before && target < before + mass) {
    e = eq;
    u64 run = before;
    for (int i = i0; i < i1; ++i) {
      run += kept(i, e);
      if (run > target) {
        sm_pick = i;
        break;
      }
    }
    a.out[row] = sm_pick;
  }
}

}  // namespace

void sample_tokens(const SampleArgs& a, cudaStream_t s) {
  if (a.rows == 0) return;
  const dim3 grid(a.rows), block(ST_THREADS);
  if (a.dtype == DT_F32) launch_pdl(sample_tokens_kernel<float>, grid, block, 0, s, a);
  else if (a.dtype == DT_F16) launch_pdl(sample_tokens_kernel<__half>, grid, block, 0, s, a);
  else launch_pdl(sample_tokens_kernel<__nv_bfloat16>, grid, block, 0, s, a);
  RT_LAUNCH_CHECK();
}

}  // namespace rt
