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
//
// A cluster of CTAs takes a row and reads it once, into shared memory.  A threshold is found with one histogram over 1024
// equal steps of 46 octaves below the maximum (counts for top_k, exact weights for top_p), whose crossing bin's few members
// are then ranked by counting; should they be too many (equal logits), the key is bisected instead.  The draw adds kept
// weights by warp, and the warp that holds the target walks its stretch.
// The row's bytes are the bound for filtered rows of large batches; summing all weights needs an exponential in 64 bits for each
// logit, about as many cycles as loading it.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>

#include "../api.h"
#include "../common/launch.h"
#include "../common/ptx.cuh"

namespace cg = cooperative_groups;

namespace rt {

namespace {

typedef unsigned long long u64;
constexpr int ST_THREADS = 512, ST_WARPS = ST_THREADS / 32;
constexpr int ST_MAX_CLUSTER = 8;
constexpr int ST_BINS = 1024;
constexpr int ST_LIST = 1536;                  // members of a crossing bin that are ranked
constexpr int ST_TABLE = 128;                  // 2^(i / 128)
constexpr double ST_ONE = 35184372088832.0;    // 2^45
constexpr float ST_OCTAVES = 46.f;             // further below the maximum weights are zero

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

struct Shared {
  double table[ST_TABLE];                      // ST_ONE 2^(i / 128)
  u64 list[ST_LIST];                           // key and ~index of a crossing bin's members
  u64 warp_a[ST_WARPS], sum[2];                // block reductions, and what the cluster reads of them
  u64 mass[ST_WARPS];                          // draw: kept weight above the cut, by warp
  unsigned ties[ST_WARPS];                     // draw: members at the cut, by warp
  union {
    struct {
      unsigned cnt[ST_BINS], lo[ST_BINS], hi[ST_BINS];
    };
    u64 list_w[ST_LIST];                       // once the crossing is known the histogram is not read again
  };
  int n_list;
  // what one CTA or thread decides for the others
  u64 found_mass, found_key;
  unsigned found_count;
  int found_bin, pick_warp;
};

// w of a logit in bins 0 .. ST_BINS - 2.  2^y = 2^(k / 128) e^r with k the nearest integer to 128 y and |r| <= ln 2 / 256,
// where the series to r^4 is off by 1e-15; adding 2^52 rounds to the integer that the low bits then hold.
struct Weigh {
  float m, bins_per;                           // maximum; bins per unit of the logit
  double m64, c;                               // 128 log2(e) / T
  const double* table;
  __device__ __forceinline__ int bin(float l) const { return l == m ? 0 : (int)fminf((m - l) * bins_per, (float)(ST_BINS - 1)); }
  __device__ __forceinline__ u64 of(float l) const {
    if (l == m) return (u64)ST_ONE;
    const double z = ((double)l - m64) * c;
    const double magic = 6755399441055744.0;   // 1.5 * 2^52
    const double t = z + magic;
    const int k = __double2loint(t);
    const double f = z - (t - magic);
    constexpr double A = 0.0054152123481245727;  // ln 2 / 128
    const double q = f * (A + f * (A * A / 2 + f * (A * A * A / 6 + f * (A * A * A * A / 24))));
    const double two = table[k & (ST_TABLE - 1)];
    const double sc = __hiloint2double(__double2hiint(two) + ((k >> 7) << 20), __double2loint(two));
    const double w = fma(sc, q, sc) + 4503599627370496.0;  // + 2^52
    return (u64)__double_as_longlong(w) & 0xfffffffffffffull;
  }
};

template <typename V, typename Op>
__device__ V warp_all(V v, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Every thread of the cluster gets the result; `turn` alternates so that one cluster barrier a call is enough.
template <typename Op>
__device__ u64 cluster_all(cg::cluster_group& cl, Shared& sm, u64 v, int& turn, Op op) {
  v = warp_all(v, op);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm.warp_a[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = warp_all(threadIdx.x < ST_WARPS ? sm.warp_a[threadIdx.x] : 0, op);  // 0 changes neither a sum nor a maximum
    if (threadIdx.x == 0) sm.sum[turn] = v;
  }
  cl.sync();
  const int nc = cl.num_blocks();
  v = cl.map_shared_rank(&sm, 0)->sum[turn];
  for (int r = 1; r < nc; ++r) v = op(v, cl.map_shared_rank(&sm, r)->sum[turn]);
  turn ^= 1;
  return v;
}

template <typename T>
__global__ void __launch_bounds__(ST_THREADS) sample_tokens_kernel(SampleArgs a, int per) {
  extern __shared__ __align__(16) unsigned char dyn[];
  Shared& sm = *reinterpret_cast<Shared*>(dyn);
  float* const slice = reinterpret_cast<float*>(dyn + sizeof(Shared));
  cg::cluster_group cl = cg::this_cluster();
  const int nc = cl.num_blocks(), rank = cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / nc;
  const int base = rank * per, n = max(0, min(per, a.vocab - base));  // this CTA's logits
  auto add = [](u64 p, u64 q) { return p + q; };
  auto larger = [](u64 p, u64 q) { return p > q ? p : q; };
  if (tid < ST_TABLE) sm.table[tid] = exp2((double)tid / ST_TABLE) * ST_ONE;
  pdl_launch_dependents();
  pdl_wait();

  // ---- the row, its maximum and the lowest index that has it
  const T* const x = (const T*)a.logits + row * a.ld + base;
  float top = -CUDART_INF_F;
  int at = 0x7fffffff;
#pragma unroll 8
  for (int i = tid; i < n; i += ST_THREADS) {
    const float l = clean(to_f(x[i]));
    slice[i] = l;
    if (l > top) {
      top = l;
      at = base + i;
    }
  }
  int turn = 0;
  const u64 best = cluster_all(cl, sm, top == -CUDART_INF_F ? 0 : ((u64)key_of(top) << 32) | (unsigned)~at, turn, larger);
  const double T_ = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
  if (best == 0 || !(T_ > 0.0)) {
    if (rank == 0 && tid == 0) a.out[row] = best == 0 ? -1 : (long long)(int)~(unsigned)best;
    cl.sync();  // no CTA leaves while another reads its shared memory
    return;
  }
  Weigh w;
  w.m = of_key((unsigned)(best >> 32));
  w.m64 = w.m;
  w.c = 1.4426950408889634074 / T_ * ST_TABLE;
  w.bins_per = (float)(1.4426950408889634074 / T_ * ((ST_BINS - 1) / ST_OCTAVES));
  w.table = sm.table;
  const int top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
  const double top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
  const double min_w = fmin(a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p, 1.0) * ST_ONE;
  const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.0;

  unsigned cut = 0;          // kept: keys above the cut, and the first `ties` that equal it
  unsigned ties = 0xffffffffu;
  auto weight = [&](float l) { return w.bin(l) < ST_BINS - 1 ? w.of(l) : 0; };

  if (by_count || by_mass) {
    // ---- histogram.  Without top_k, weights below (1 - top_p) / vocab cannot be where top_p is reached: all of them together weigh less.
    const u64 floor_w = by_count || !(top_p > 0.0) ? 0 : (u64)((1.0 - top_p) / a.vocab * ST_ONE);
    for (int b = tid; b < ST_BINS; b += ST_THREADS) sm.cnt[b] = sm.lo[b] = sm.hi[b] = 0;
    if (tid == 0) sm.n_list = 0;
    __syncthreads();
    u64 total = 0;
    for (int i = tid; i < n; i += ST_THREADS) {
      const float l = slice[i];
      const int b = w.bin(l);
      if (b == ST_BINS - 1) continue;
      if (by_count) atomicAdd(&sm.cnt[b], 1u);
      if (by_mass) {
        const u64 v = w.of(l);
        total += v;
        if (v > floor_w) {
          const unsigned low = (unsigned)v, old = atomicAdd(&sm.lo[b], low);
          const unsigned high = (unsigned)(v >> 32) + (old + low < old);
          if (high) atomicAdd(&sm.hi[b], high);
        }
      }
    }
    if (by_mass) total = cluster_all(cl, sm, total, turn, add);
    else cl.sync();

    // the first bin at which the running sum over the cluster's histograms reaches `want`, and the sum before it; -1: none
    auto crossing = [&](bool mass, u64 want, u64* before) {
      u64 v[ST_BINS / ST_THREADS], mine = 0;
      for (int e = 0; e < ST_BINS / ST_THREADS; ++e) {
        const int b = tid * (ST_BINS / ST_THREADS) + e;
        v[e] = 0;
        for (int r = 0; r < nc; ++r) {
          const Shared* o = cl.map_shared_rank(&sm, r);
          v[e] += mass ? ((u64)o->hi[b] << 32) + o->lo[b] : (u64)o->cnt[b];
        }
        mine += v[e];
      }
      u64 run = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      __syncthreads();
      if (lane == 31) sm.warp_a[warp] = run;
      if (tid == 0) sm.found_bin = -1;
      __syncthreads();
      run -= mine;
      for (int k = 0; k < warp; ++k) run += sm.warp_a[k];
      for (int e = 0; e < ST_BINS / ST_THREADS; ++e) {
        if (run < want && run + v[e] >= want) {
          sm.found_bin = tid * (ST_BINS / ST_THREADS) + e;
          sm.found_mass = run;
        }
        run += v[e];
      }
      __syncthreads();
      *before = sm.found_mass;
      return sm.found_bin;
    };
    // the members of a bin, in CTA 0's list; returns how many there are
    auto gather = [&](int bin) {
      Shared* const first = cl.map_shared_rank(&sm, 0);
      for (int i = tid; i < n; i += ST_THREADS) {
        const float l = slice[i];
        if (w.bin(l) != bin) continue;
        const int k = atomicAdd(&first->n_list, 1);
        if (k < ST_LIST) first->list[k] = ((u64)key_of(l) << 32) | (unsigned)~(base + i);
      }
      cl.sync();
      return first->n_list;
    };
    // sum over keys >= t: how many, or their weight
    auto above = [&](unsigned t, bool mass) {
      u64 v = 0;
      for (int i = tid; i < n; i += ST_THREADS) {
        const float l = slice[i];
        if (key_of(l) >= t) v += mass ? weight(l) : 1;
      }
      return cluster_all(cl, sm, v, turn, add);
    };
    auto bisect = [&](u64 want, bool mass) {  // largest key t with above(t) >= want
      unsigned t = 0;
      for (int b = 31; b >= 0; --b)
        if (above(t | (1u << b), mass) >= want) t |= 1u << b;
      return t;
    };

    int k_bin = -1;
    if (by_count) {
      u64 before;
      k_bin = crossing(false, (u64)top_k, &before);
      if (k_bin >= 0) {  // else every possible token is among the first top_k
        const int members = gather(k_bin);
        if (members <= ST_LIST) {
          if (rank == 0) {
            const unsigned r = (unsigned)(top_k - before);  // 1 .. members
            for (int i = tid; i < members; i += ST_THREADS) {
              const u64 e = sm.list[i];
              unsigned ahead = 0, over = 0;
              for (int k = 0; k < members; ++k) {
                ahead += sm.list[k] > e;
                over += (unsigned)(sm.list[k] >> 32) > (unsigned)(e >> 32);
              }
              if (ahead == r - 1) {
                sm.found_key = e >> 32;
                sm.found_count = r - over;
              }
            }
          }
          cl.sync();
          const Shared* const first = cl.map_shared_rank(&sm, 0);
          cut = (unsigned)first->found_key;
          ties = first->found_count;
        } else {
          cut = bisect((u64)top_k, false);
          ties = (unsigned)((u64)top_k - (cut == 0xffffffffu ? 0 : above(cut + 1, false)));
        }
        if (by_mass) total = (cut == 0xffffffffu ? 0 : above(cut + 1, true)) + ties * weight(of_key(cut));
      }
    }
    if (by_mass) {
      const double part = ceil((top_p > 0.0 ? top_p : 0.0) * (double)total);
      const u64 want = part >= 1.0 ? (part < (double)total ? (u64)part : total) : 1;
      u64 before;
      const int bin = crossing(true, want, &before);
      int members = ST_LIST + 1;
      if (bin >= 0) {
        if (k_bin >= 0) {  // the list is used again
          cl.sync();
          if (tid == 0) sm.n_list = 0;
          cl.sync();
        }
        members = gather(bin);
      }
      unsigned new_cut, new_ties;
      if (members <= ST_LIST) {
        if (rank == 0) {
          for (int i = tid; i < members; i += ST_THREADS) sm.list_w[i] = weight(of_key((unsigned)(sm.list[i] >> 32)));
          __syncthreads();
          for (int i = tid; i < members; i += ST_THREADS) {
            const u64 e = sm.list[i];
            u64 run = before;
            unsigned equal = 0;
            for (int k = 0; k < members; ++k)
              if (sm.list[k] > e) {
                run += sm.list_w[k];
                equal += (unsigned)(sm.list[k] >> 32) == (unsigned)(e >> 32);
              }
            if (run < want && run + sm.list_w[i] >= want) {  // the last one that is kept
              sm.found_key = e >> 32;
              sm.found_count = equal + 1;
            }
          }
        }
        cl.sync();
        const Shared* const first = cl.map_shared_rank(&sm, 0);
        new_cut = (unsigned)first->found_key;
        new_ties = first->found_count;
      } else {
        new_cut = bisect(want, true);
        const u64 over = new_cut == 0xffffffffu ? 0 : above(new_cut + 1, true), v = weight(of_key(new_cut));
        new_ties = v ? (unsigned)((want - over + v - 1) / v) : 1;
      }
      if (new_cut > cut || (new_cut == cut && new_ties < ties)) {
        cut = new_cut;
        ties = new_ties;
      }
    }
  }

  // ---- draw: a warp's stretch is contiguous
  const int seg = (per + ST_THREADS - 1) / ST_THREADS * 32;
  const int s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
  const u64 cut_w = cut ? weight(of_key(cut)) : 0;
  const bool cut_in = cut_w && (of_key(cut) == w.m || (double)cut_w >= min_w);
  auto over_cut = [&](float l) -> u64 {  // weight of a key above the cut, 0 where min_p takes it out
    if (key_of(l) <= cut) return 0;
    const u64 v = weight(l);
    return l == w.m || (double)v >= min_w ? v : 0;
  };
  u64 mass = 0;
  unsigned eq = 0;
  for (int i = s0 + lane; i < s1; i += 32) {
    const float l = slice[i];
    mass += over_cut(l);
    eq += key_of(l) == cut;
  }
  mass = warp_all(mass, add);
  eq = warp_all(eq, [](unsigned p, unsigned q) { return p + q; });
  if (lane == 0) {
    sm.mass[warp] = mass;
    sm.ties[warp] = eq;
  }
  if (tid == 0) sm.pick_warp = -1;
  cl.sync();
  double u = a.uniform_f64 ? ((const double*)a.uniform)[row] : (double)((const float*)a.uniform)[row];
  u = u > 0.0 ? u : 0.0;
  if (warp == 0) {
    // all stretches of the row in order, ST_MAX_CLUSTER * ST_WARPS / 32 a lane
    constexpr int PER = ST_MAX_CLUSTER * ST_WARPS / 32;
    u64 m[PER], all = 0;
    unsigned t[PER], before_t = 0;
    for (int e = 0; e < PER; ++e) {
      const int k = lane * PER + e;
      const Shared* o = cl.map_shared_rank(&sm, k / ST_WARPS < nc ? k / ST_WARPS : 0);
      m[e] = k / ST_WARPS < nc ? o->mass[k % ST_WARPS] : 0;
      t[e] = k / ST_WARPS < nc ? o->ties[k % ST_WARPS] : 0;
      before_t += t[e];
    }
    unsigned run_t = before_t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, run_t, o);
      if (lane >= o) run_t += up;
    }
    run_t -= before_t;
    unsigned first_t[PER];
    for (int e = 0; e < PER; ++e) {
      first_t[e] = run_t;
      const unsigned in = run_t < ties ? min(t[e], ties - run_t) : 0;
      if (cut_in) m[e] += in * cut_w;
      run_t += t[e];
      all += m[e];
    }
    u64 run = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    const u64 target = __umul64hi(u < 1.0 ? (u64)(u * 18446744073709551616.0) : ~0ull, __shfl_sync(0xffffffffu, run, 31));
    run -= all;
    for (int e = 0; e < PER; ++e) {
      const int k = lane * PER + e;
      if (target >= run && target < run + m[e] && k / ST_WARPS == rank) {
        sm.pick_warp = k % ST_WARPS;
        sm.found_mass = target - run;
        sm.found_count = first_t[e];
      }
      run += m[e];
    }
  }
  __syncthreads();
  if (sm.pick_warp == warp) {
    u64 left = sm.found_mass;
    unsigned tie = sm.found_count;
    for (int i0 = s0; i0 < s1; i0 += 32) {
      const int i = i0 + lane;
      const float l = i < s1 ? slice[i] : -CUDART_INF_F;
      const bool equal = i < s1 && key_of(l) == cut;
      const unsigned eqs = __ballot_sync(0xffffffffu, equal);
      u64 v = i < s1 ? over_cut(l) : 0;
      if (equal && cut_in && tie + __popc(eqs & ((1u << lane) - 1)) < ties) v = cut_w;
      tie += __popc(eqs);
      if (!__any_sync(0xffffffffu, v != 0)) continue;
      u64 run = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, run > left);
      if (hit) {
        if (lane == __ffs(hit) - 1) a.out[row] = base + i;
        break;
      }
      left -= __shfl_sync(0xffffffffu, run, 31);
    }
  }
  cl.sync();  // no CTA leaves while another reads its shared memory
}

template <typename T>
void launch(const SampleArgs& a, cudaStream_t s) {
  // Smallest cluster whose slices let three CTAs share an SM; more CTAs a row while the batch leaves SMs idle.
  int nc = 1;
  while (nc < ST_MAX_CLUSTER && (a.vocab + nc - 1) / nc > 8192) nc *= 2;
  while (nc < ST_MAX_CLUSTER && (long long)a.rows * nc * 2 <= sm_count(current_device()) && a.vocab / nc > 2048) nc *= 2;
  const int per = (a.vocab + nc - 1) / nc;
  const int smem = (int)sizeof(Shared) + per * 4;
  static int allowed[64] = {0};
  const int dev = current_device();
  if (smem > allowed[dev]) {
    RT_CUDA_CHECK(cudaFuncSetAttribute((const void*)sample_tokens_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    allowed[dev] = smem;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * nc));
  cfg.blockDim = dim3(ST_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = nc;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  RT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, sample_tokens_kernel<T>, a, per));
  RT_LAUNCH_CHECK();
}

}  // namespace

void sample_tokens(const SampleArgs& a, cudaStream_t s) {
  if (a.rows == 0) return;
  RT_CHECK(a.vocab >= 1 && a.vocab <= 262144 && a.rows < (1 << 28), "sample_tokens: unsupported sizes");
  if (a.dtype == DT_F32) launch<float>(a, s);
  else if (a.dtype == DT_F16) launch<__half>(a, s);
  else launch<__nv_bfloat16>(a, s);
}

}  // namespace rt
