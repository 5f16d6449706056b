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
// A cluster of CTAs takes a row and reads it once, into shared memory.  A threshold is found by histograms (counts for top_k,
// exact weights for top_p): over 384 equal steps of 46 octaves below the maximum, then over 384 steps of the one where the
// sum crosses; the few members of that step are ranked by a warp, and should they be too many (equal logits) the histograms
// go on over their keys.  Members of a crossing step are queued by the one pass that compares floats to find them, and only the queue is
// looked at again.  The draw needs each CTA's kept weight, which its part of the first histogram and the queue give; then only the
// CTA that holds the target adds by warp, by parts of a warp's stretch, and walks.
// A top_k whose candidates fit one CTA (384) is finished there, all filters and the draw (1 x 32000, top_k 50, top_p 0.9: 10 us, 21 without).
// Where all weights are summed (top_p or no filter) no unit is full: 256 x 128256 with top_p 0.95 take 258 us, 20 by their bytes, with
// issue slots 57 % busy and the FP64 pipe 12 % (a 64-bit exponential is 18 instructions a logit); 2048 CTAs, three an SM, go in 4.6
// waves through load, barrier, pass, barrier, one after the other.
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
constexpr int ST_THREADS = 384, ST_WARPS = ST_THREADS / 32;  // three CTAs an SM beside 64 KB slices
constexpr int ST_MAX_CLUSTER = 8;
constexpr int ST_BINS = ST_THREADS;            // a bin a thread where sums over them are formed
constexpr int ST_FEW = ST_THREADS;             // candidates that one CTA finishes, a thread each
constexpr int ST_LIST = 64;                    // members of a step that a warp ranks
constexpr int ST_QUEUE = 512;                  // members of a step that a CTA keeps at hand
constexpr int ST_TABLE = 128;                  // 2^(i / 128)
constexpr double ST_ONE = 35184372088832.0;    // 2^45
constexpr double ST_OCTAVES = 46.0;            // further below the maximum weights are zero

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float clean(float l) { return fmaxf(l, -CUDART_INF_F); }  // NaN counts as minus infinity
__device__ __forceinline__ unsigned key_of(float l) {  // in the order of the values; -0 and 0 get one key
  const unsigned b = __float_as_uint(l + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct alignas(16) Shared {
  double table[ST_TABLE];                      // ST_ONE 2^(i / 128)
  u64 part[2][ST_WARPS];                       // reductions by warp, used in turn
  u64 mass[ST_WARPS], fine_mass[ST_WARPS];     // draw: kept weight above the cut, by warp
  unsigned ties[ST_WARPS], fine_ties[ST_WARPS];  // draw: members at the cut, by warp
  struct {
    unsigned lo[ST_BINS], hi[ST_BINS];         // counts in lo, weights in both
  } hist[2];                                   // the first histogram, and finer ones; of the first CTA also the few of a small top_k
  unsigned list[2][ST_LIST];                   // keys of a finer step's members, for top_k and for top_p (the first CTA's)
  float queue[ST_QUEUE];                       // this CTA's members of the crossing step
  int n_list[2], n_queue;
  u64 cta_mass;                                // draw: of the whole CTA
  unsigned cta_ties;
  // what one thread finds for its CTA
  u64 found_mass, found_upto;
  unsigned found_key;
  int found_bin;
};

// w of a logit l with steps_below(l) < ST_BINS - 1.  2^y = 2^(k / 128) e^r with k the nearest integer to 128 y and
// |r| <= ln 2 / 256, where the series to r^4 is off by 1e-15; adding 2^52 rounds to the integer that the low bits then hold.
struct Weigh {
  float m, per;                                // maximum; histogram steps per unit of the logit
  double m64, c, step;                         // 128 log2(e) / T; 1 / per
  const double* table;
  // steps below the maximum, monotone in l; 0 for the maximum itself, also where a product with infinity is none
  __device__ __forceinline__ float steps_below(float l) const { return fmaxf((m - l) * per, 0.f); }
  __device__ __forceinline__ bool possible(float l) const { return steps_below(l) < ST_BINS - 1; }
  template <int N> __device__ __forceinline__ void of(const float (&l)[N], u64 (&w)[N]) const {  // side by side: the chain is long
    constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52
    constexpr double A = 0.0054152123481245727;   // ln 2 / 128
    double f[N], sc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = ((double)l[e] - m64) * c;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const double t = f[e] + MAGIC;
      const int k = __double2loint(t);
      f[e] -= t - MAGIC;
      const double two = table[k & (ST_TABLE - 1)];
      static_assert(ST_TABLE == 128, "the exponent's share of k, moved from bit 7 to bit 20");
      sc[e] = __hiloint2double(__double2hiint(two) + (k & ~(ST_TABLE - 1)) * (1 << 13), __double2loint(two));
    }
    double q[N];
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = fma(f[e], A * A * A * A / 24, A * A * A / 6);
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = fma(f[e], q[e], A * A / 2);
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = f[e] * fma(f[e], q[e], A);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      w[e] = (u64)__double_as_longlong(fma(sc[e], q[e], sc[e]) + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52
    }
  }
  __device__ __forceinline__ u64 of(float l) const {
    const float x[1] = {l};
    u64 v[1];
    of(x, v);
    return v[0];
  }
  __device__ __forceinline__ u64 operator()(float l) const { return possible(l) ? of(l) : 0; }
  // floats around the logits that lie `steps` below the maximum: rounding moves steps_below by 5e-5 at most
  __device__ __forceinline__ float surely_below(double steps) const { return __double2float_rd(m64 - (steps + 5e-4) * step); }
  __device__ __forceinline__ float surely_above(double steps) const { return steps <= 0 ? CUDART_INF_F : __double2float_ru(m64 - (steps - 5e-4) * step); }
};

struct Add {
  template <typename V> __device__ __forceinline__ V operator()(V p, V q) const { return p + q; }
};
struct Larger {
  template <typename V> __device__ __forceinline__ V operator()(V p, V q) const { return p > q ? p : q; }
};

template <typename V, typename Op>
__device__ __forceinline__ V warp_all(V v, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_before(V v, int lane) {  // sum over the lanes before this one
  V run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  return run - v;
}

// Every thread of the cluster gets the result (0 must change nothing); `turn` alternates, so one cluster barrier a call is enough.
template <typename Op>
__device__ __forceinline__ u64 cluster_all(cg::cluster_group& cl, int nc, Shared& sm, u64 v, int& turn, Op op) {
  v = warp_all(v, op);
  if ((threadIdx.x & 31) == 0) sm.part[turn][threadIdx.x >> 5] = v;
  cl.sync();
  constexpr int PER = (ST_MAX_CLUSTER * ST_WARPS + 31) / 32;
  u64 got[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int k = (threadIdx.x & 31) + 32 * e;
    got[e] = k < nc * ST_WARPS ? cl.map_shared_rank(&sm, k / ST_WARPS)->part[turn][k % ST_WARPS] : 0;
  }
  v = got[0];
#pragma unroll
  for (int e = 1; e < PER; ++e) v = op(v, got[e]);
  turn ^= 1;
  return warp_all(v, op);
}

// The CTA's n logits to shared memory, cleaned: logit i at slice[pad + i], minus infinity on either side up to whole groups of
// four; returns this thread's largest.  Rows may start anywhere: single values up to a 16-byte boundary (logit `head`),
// 16 bytes at a time from there on; `pad` puts those on 16 bytes of shared memory too.
template <typename T>
__device__ __forceinline__ float load_slice(const T* x, float* slice, int n, int head, int pad, int quads) {
  constexpr int PER = 16 / sizeof(T);
  float top = -CUDART_INF_F;
  const int vecs = n > head ? (n - head) / PER : 0, tail = n > head ? head + vecs * PER : n;
  const uint4* const v = reinterpret_cast<const uint4*>(x + head);
#pragma unroll 4
  for (int i = threadIdx.x; i < vecs; i += ST_THREADS) {
    const uint4 r = __ldcs(v + i);
    const T* const e = reinterpret_cast<const T*>(&r);
    float f[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      f[k] = clean(to_f(e[k]));
      top = fmaxf(top, f[k]);
    }
#pragma unroll
    for (int k = 0; k < PER; k += 4) *reinterpret_cast<float4*>(slice + pad + head + i * PER + k) = make_float4(f[k], f[k + 1], f[k + 2], f[k + 3]);
  }
  // what is left at both ends, a thread each: pad and head, then tail and pad
  const int front = pad + min(head, n), rest = 4 * quads - pad - tail;
  if ((int)threadIdx.x < front + rest) {
    const int j = (int)threadIdx.x < front ? (int)threadIdx.x : pad + tail + (int)threadIdx.x - front;
    const int i = j - pad;
    const float l = i >= 0 && i < n ? clean(to_f(x[i])) : -CUDART_INF_F;
    slice[j] = l;
    top = fmaxf(top, l);
  }
  return top;
}

template <typename T>
__global__ void __launch_bounds__(ST_THREADS, 3) sample_tokens_kernel(SampleArgs a, int per) {
  extern __shared__ __align__(16) unsigned char dyn[];
  Shared& sm = *reinterpret_cast<Shared*>(dyn);
  float* const slice = reinterpret_cast<float*>(dyn + sizeof(Shared));
  const float4* const slice4 = reinterpret_cast<const float4*>(slice);
  cg::cluster_group cl = cg::this_cluster();
  const int nc = cl.num_blocks(), rank = cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / nc;
  const int base = rank * per, n = max(0, min(per, a.vocab - base));  // this CTA's logits
  if (tid < ST_TABLE) sm.table[tid] = exp2((double)tid / ST_TABLE) * ST_ONE;
  if (tid < 2) sm.n_list[tid] = 0;
  pdl_launch_dependents();
  pdl_wait();

  // ---- the row and its maximum
  const T* const x = (const T*)a.logits + row * a.ld + base;
  const int head = (int)((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)), pad = (4 - head % 4) % 4;
  const int quads = (pad + n + 3) / 4;
  const float top = load_slice(x, slice, n, head, pad, quads);
  int turn = 0;
  const unsigned best = (unsigned)cluster_all(cl, nc, sm, top == -CUDART_INF_F ? 0 : key_of(top), turn, Larger());
  const double T_ = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
  Weigh w;
  w.m = of_key(best);
  if (best == 0 || !(T_ > 0.0)) {  // no possible token, or the most likely one: the lowest index that holds the maximum
    u64 first = 0;
    if (best != 0)
      for (int j = tid; j < 4 * quads && !first; j += ST_THREADS)
        if (slice[j] == w.m) first = (unsigned)~(base + j - pad);
    first = cluster_all(cl, nc, sm, first, turn, Larger());
    if (rank == 0 && tid == 0) a.out[row] = best == 0 ? -1 : (long long)(int)~(unsigned)first;
    cl.sync();  // no CTA leaves while another reads its shared memory
    return;
  }
  if (w.m == CUDART_INF_F) {  // such logits share all the weight: the row becomes 0 for them and minus infinity elsewhere
    __syncthreads();
    for (int j = tid; j < 4 * quads; j += ST_THREADS) slice[j] = slice[j] == CUDART_INF_F ? 0.f : -CUDART_INF_F;
    w.m = 0.f;
    __syncthreads();
  }
  w.m64 = w.m;
  w.c = fmin(1.4426950408889634074 / T_ * ST_TABLE, 1e300);
  w.per = fmaxf((float)(1.4426950408889634074 / T_ * ((ST_BINS - 1) / ST_OCTAVES)), 1.17549435e-38f);  // times infinity it stays infinity
  w.step = 1.0 / (double)w.per;
  w.table = sm.table;
  const int top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
  const double top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
  const double min_p = fmax(0.0, fmin(a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p, 1.0));
  const u64 min_w = (u64)ceil(min_p * ST_ONE);
  // steps down to the weight p of the maximum's, a hundredth too many at most
  auto steps_to = [](double p) { return fminf(fmaxf(-log2f((float)p) * (float)((ST_BINS - 1) / ST_OCTAVES), 0.f) + 0.01f, ST_BINS - 1.f); };
  const float min_steps = steps_to(min_p);
  const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.0;
  auto wanted = [&](u64 total) -> u64 {  // the mass that top_p asks for, a part of the first token at least
    const double some = ceil((top_p > 0.0 ? top_p : 0.0) * (double)total);
    return some >= 1.0 ? (some < (double)total ? (u64)some : total) : 1;
  };
  auto fraction = [&]() -> u64 {  // the row's number in 2^-64
    double u = a.uniform_f64 ? ((const double*)a.uniform)[row] : (double)((const float*)a.uniform)[row];
    u = u > 0.0 ? u : 0.0;
    return u < 1.0 ? (u64)(u * 18446744073709551616.0) : ~0ull;
  };
  // f(l) for this thread's logits l >= least, where few are
  auto each = [&](float least, auto f) {
    for (int q = tid; q < quads; q += ST_THREADS) {
      const float4 l = slice4[q];
      if (fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w)) < least) continue;
      if (l.x >= least) f(l.x);
      if (l.y >= least) f(l.y);
      if (l.z >= least) f(l.z);
      if (l.w >= least) f(l.w);
    }
  };
  // the least float from `low` to the maximum that is kept by a test that larger ones pass too; 32 at a time, in every warp
  auto least_that = [&](float low, auto passes) {
    unsigned k_lo = key_of(low), k_hi = key_of(w.m);
    while (k_lo < k_hi) {
      const unsigned step = (k_hi - k_lo + 31) / 32, k = min(k_hi, k_lo + lane * step);
      const unsigned ok = __ballot_sync(0xffffffffu, passes(of_key(k)));
      const int at = ok ? __ffs(ok) - 1 : 32;
      if (at < 32) k_hi = min(k_hi, k_lo + at * step);
      if (at > 0) k_lo = min(k_hi, k_lo + (at - 1) * step + 1);
    }
    return of_key(k_hi);
  };
  const float least_possible = least_that(w.surely_below(ST_BINS - 1), [&](float l) { return w.possible(l); });

  float cut = -CUDART_INF_F;  // kept: logits above the cut, and the first `ties` that equal it
  unsigned ties = 0;
  // f(l) for the members of a step of the first histogram that are in this CTA
  int step_bin = -1;
  auto members = [&](auto f) {
    if (sm.n_queue <= ST_QUEUE) {
      for (int i = tid; i < sm.n_queue; i += ST_THREADS) f(sm.queue[i]);
    } else {
      each(w.surely_below(step_bin + 1), [&](float l) {
        const float t = w.steps_below(l);
        if (t < ST_BINS - 1 && (int)t == step_bin) f(l);
      });
    }
  };
  if (by_count || by_mass) {
    auto clear = [&](int h) {
      sm.hist[h].lo[tid] = sm.hist[h].hi[tid] = 0;
      __syncthreads();
    };
    auto put = [&](int h, int b, u64 v) {
      const unsigned low = (unsigned)v, old = atomicAdd(&sm.hist[h].lo[b], low);
      const unsigned high = (unsigned)(v >> 32) + (old + low < old);
      if (high) atomicAdd(&sm.hist[h].hi[b], high);
    };
    // The first bin at which the running sum over the cluster's histograms h reaches `want`, -1: none.  The sum before it is added to
    // `before`.
    auto crossing = [&](int h, bool mass, u64 want, u64& before) {
      unsigned lo[ST_MAX_CLUSTER], hi[ST_MAX_CLUSTER];
#pragma unroll
      for (int r = 0; r < ST_MAX_CLUSTER; ++r) {
        const Shared* const o = cl.map_shared_rank(&sm, r < nc ? r : 0);
        lo[r] = r < nc ? o->hist[h].lo[tid] : 0;
        hi[r] = r < nc && mass ? o->hist[h].hi[tid] : 0;
      }
      u64 v = 0;
#pragma unroll
      for (int r = 0; r < ST_MAX_CLUSTER; ++r) v += ((u64)hi[r] << 32) + lo[r];
      u64 run = warp_before(v, lane);
      if (lane == 31) sm.mass[warp] = run + v;
      if (tid == 0) sm.found_bin = -1;
      __syncthreads();
      run += before + warp_all(lane < warp ? sm.mass[lane] : 0, Add());
      if (run < want && run + v >= want) {
        sm.found_bin = tid;
        sm.found_mass = run;
        sm.found_upto = run + v;
      }
      __syncthreads();
      const int bin = sm.found_bin;
      if (bin >= 0) before = sm.found_mass;
      __syncthreads();
      return bin;
    };
    // The logit at which the sum reaches `want`, a member of step `bin` of the first histogram; `before` becomes the sum over
    // larger logits.
    auto narrow = [&](bool mass, u64 want, int bin, u64& before) {
      auto sub_step = [&](float l) { return (int)((w.steps_below(l) - bin) * ST_BINS); };
      step_bin = bin;
      const float most = w.surely_above(bin);
      if (tid == 0) sm.n_queue = 0;
      clear(1);
      each(w.surely_below(bin + 1), [&](float l) {
        const float t = w.steps_below(l);
        if (l > most || !(t < ST_BINS - 1) || (int)t != bin) return;
        const int k = atomicAdd(&sm.n_queue, 1);
        if (k < ST_QUEUE) sm.queue[k] = l;
      });
      __syncthreads();
      members([&](float l) {
        if (mass) put(1, sub_step(l), w.of(l));
        else atomicAdd(&sm.hist[1].lo[sub_step(l)], 1u);
      });
      cl.sync();
      const int sub = crossing(1, mass, want, before);
      Shared* const first = cl.map_shared_rank(&sm, 0);
      const int which = mass ? 1 : 0;
      members([&](float l) {
        if (sub_step(l) != sub) return;
        const int k = atomicAdd(&first->n_list[which], 1);
        if (k < ST_LIST) first->list[which][k] = key_of(l);
      });
      cl.sync();
      const int found = first->n_list[which];
      if (found <= ST_LIST) {
        if (warp == 0) {
          // a lane weighs up to two members against all
          unsigned k[2];
          u64 v[2], over[2] = {before, before}, eq[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            k[e] = lane + 32 * e < found ? first->list[which][lane + 32 * e] : 0;
            v[e] = k[e] == 0 ? 0 : mass ? w(of_key(k[e])) : 1;
          }
          for (int j = 0; j < found; ++j) {
            const unsigned kj = __shfl_sync(0xffffffffu, j < 32 ? k[0] : k[1], j & 31);
            const u64 vj = __shfl_sync(0xffffffffu, j < 32 ? v[0] : v[1], j & 31);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (kj > k[e]) over[e] += vj;
              if (kj == k[e]) eq[e] += vj;
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (k[e] != 0 && over[e] < want && over[e] + eq[e] >= want) {
              sm.found_key = k[e];  // equal members write the same
              sm.found_mass = over[e];
            }
        }
        __syncthreads();
        before = sm.found_mass;
        return of_key(sm.found_key);
      }
      // Many members in so narrow a step are equal ones, or nearly so: histograms over their keys, until a step is one key.
      unsigned k_hi = min(key_of(w.m), key_of(most)), k_lo = key_of(w.surely_below(bin + 1));
      while (true) {
        int shift = 0;
        while (((k_hi - k_lo) >> shift) >= ST_BINS) ++shift;
        cl.sync();  // the last histogram has been read
        clear(1);
        members([&](float l) {
          const unsigned k = key_of(l);
          if (k < k_lo || k > k_hi || sub_step(l) != sub) return;
          if (mass) put(1, (k_hi - k) >> shift, w.of(l));
          else atomicAdd(&sm.hist[1].lo[(k_hi - k) >> shift], 1u);
        });
        cl.sync();
        const int s = crossing(1, mass, want, before);
        k_hi -= (unsigned)max(s, 0) << shift;  // a sum that reaches `want` among these members does so in one of their steps
        if (shift == 0) return of_key(k_hi);
        k_lo = max(k_lo, k_hi - ((1u << shift) - 1));
      }
    };

    u64 total = 0, before = 0;
    bool counted = false;
    clear(0);
    if (by_count) {
      for (int q = tid; q < quads; q += ST_THREADS) {
        const float4 l4 = slice4[q];
        const float l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (l[e] >= least_possible) atomicAdd(&sm.hist[0].lo[(int)w.steps_below(l[e])], 1u);
      }
      cl.sync();
      const int bin = crossing(0, false, (u64)top_k, before);
      if (bin >= 0 && sm.found_upto <= ST_FEW) {
        // A small top_k: the first CTA gets everything down to the crossing step and finishes alone, a candidate a thread.  Two
        // loops over the candidates (what is ahead in the order, what is before in the vocabulary) take the place of all further passes.
        Shared* const first = cl.map_shared_rank(&sm, 0);
        u64* const put_few = reinterpret_cast<u64*>(&first->hist[1]);
        const float down_to = w.surely_below(bin + 1);
        for (int q = tid; q < quads; q += ST_THREADS) {
          const float4 l4 = slice4[q];
          const float l[4] = {l4.x, l4.y, l4.z, l4.w};
          if (fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) < down_to) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (l[e] >= fmaxf(down_to, least_possible) && (int)w.steps_below(l[e]) <= bin)
              put_few[atomicAdd(&first->n_list[0], 1)] = ((u64)key_of(l[e]) << 32) | (unsigned)~(base + 4 * q + e - pad);
        }
        cl.sync();
        if (rank == 0) {
          const u64* const few = reinterpret_cast<const u64*>(&sm.hist[1]);
          u64* const few_w = reinterpret_cast<u64*>(&sm.hist[0]);
          const int count = sm.n_list[0];
          auto block_sum = [&](u64 v) {
            v = warp_all(v, Add());
            __syncthreads();
            if (lane == 0) sm.mass[warp] = v;
            __syncthreads();
            return warp_all(lane < ST_WARPS ? sm.mass[lane] : 0, Add());
          };
          const u64 mine = tid < count ? few[tid] : 0;
          u64 v = mine ? w.of(of_key((unsigned)(mine >> 32))) : 0;
          few_w[tid] = v;
          __syncthreads();
          int ahead = 0;
          u64 run = 0;
#pragma unroll 4
          for (int k = 0; k < count; ++k)
            if (few[k] > mine) {
              ++ahead;
              run += few_w[k];
            }
          bool keep = mine && ahead < top_k && v >= min_w;
          if (by_mass) {
            const u64 want = wanted(block_sum(ahead < top_k ? v : 0));  // by all threads
            keep = keep && run < want;
          }
          v = keep ? v : 0;
          const u64 all = block_sum(v);
          few_w[tid] = v;
          __syncthreads();
          u64 from = 0;
#pragma unroll 4
          for (int k = 0; k < count; ++k) from += (unsigned)few[k] > (unsigned)mine ? few_w[k] : 0;
          const u64 target = __umul64hi(fraction(), all);
          if (keep && target >= from && target < from + v) a.out[row] = (long long)(int)~(unsigned)mine;
        }
        cl.sync();  // no CTA leaves while another reads its shared memory
        return;
      }
      if (bin >= 0) {  // else every possible token is among the first top_k
        cut = narrow(false, (u64)top_k, bin, before);
        ties = (unsigned)((u64)top_k - before);
        counted = true;
      }
    }
    if (by_mass) {
      // Without top_k, weights below (1 - top_p) / (2 vocab) cannot be where top_p is reached: all of them together weigh less than the rest.
      const double floor_p = by_count ? 0.0 : (1.0 - fmax(top_p, 0.0)) / a.vocab * 0.5;
      const float floor_l = w.surely_below(steps_to(floor_p));
      if (by_count) {
        if (!counted) cl.sync();  // the counts have been read
        clear(0);
      }
      const float above = counted ? of_key(key_of(cut) + 1) : least_possible, put_from = fmaxf(fmaxf(cut, least_possible), floor_l);
      for (int q = tid; q < quads; q += ST_THREADS) {
        const float4 l4 = slice4[q];
        const float l[4] = {l4.x, l4.y, l4.z, l4.w};
        if (fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) < fmaxf(cut, least_possible)) continue;
        u64 v[4];
        w.of(l, v);
        unsigned old[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (l[e] >= above) total += v[e];
          old[e] = l[e] >= put_from ? atomicAdd(&sm.hist[0].lo[(int)w.steps_below(l[e])], (unsigned)v[e]) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned high = (unsigned)(v[e] >> 32) + (old[e] + (unsigned)v[e] < old[e]);
          if (l[e] >= put_from && high) atomicAdd(&sm.hist[0].hi[(int)w.steps_below(l[e])], high);
        }
      }
      total = cluster_all(cl, nc, sm, total, turn, Add());
      if (counted) total += ties * w(cut);
      const u64 want = wanted(total);
      before = 0;
      const int bin = crossing(0, true, want, before);
      if (bin >= 0) {  // else every token above the cut is needed
        const float at = narrow(true, want, bin, before);
        const u64 v = w(at);
        const unsigned now = (unsigned)((want - before + v - 1) / v);
        if (at > cut || now < ties) {
          cut = at;
          ties = now;
        }
      }
    }
  }

  // ---- draw.  A warp's stretch is contiguous; the one that holds the target is cut into a part for each warp of its CTA, and the
  // part that holds it is walked.
  const float least = min_p > 0.0 ? fmaxf(least_possible, least_that(fmaxf(least_possible, w.surely_below(min_steps)), [&](float l) { return w.of(l) >= min_w; }))
                                  : least_possible;
  const u64 cut_w = ties && cut >= least ? w.of(cut) : 0;
  const bool cut_in = cut_w != 0;
  const float lower = fmaxf(least, ties ? of_key(key_of(cut) + 1) : least);  // kept: l >= lower, and the cut's
  auto stretch = [&](int j0, int j1, u64* mass, unsigned* equal) {  // whole groups of four
    u64 m = 0;
    unsigned eq = 0;
    for (int q = j0 / 4 + lane; q < j1 / 4; q += 32) {
      const float4 l4 = slice4[q];
      const float l[4] = {l4.x, l4.y, l4.z, l4.w};
      const float top4 = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3]));
      if (cut_in) eq += (l[0] == cut) + (l[1] == cut) + (l[2] == cut) + (l[3] == cut);
      if (top4 < lower) continue;
      u64 v[4];
      w.of(l, v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (l[e] >= lower) m += v[e];
    }
    m = warp_all(m, Add());
    eq = warp_all(eq, Add());
    if (lane == 0) {
      *mass = m;
      *equal = eq;
    }
  };
  const int end = 4 * quads, seg = ((per + 3 + ST_WARPS - 1) / ST_WARPS + 127) / 128 * 128;
  // steps of the first histogram that are kept whole: those above the cut's, whose members are queued; none where min_p cuts higher
  const int whole = by_mass && cut_in ? (int)w.steps_below(cut) : 0;
  if (whole > 0) {
    u64 m = tid < whole ? ((u64)sm.hist[0].hi[tid] << 32) + sm.hist[0].lo[tid] : 0;
    unsigned eq = 0;
    members([&](float l) {
      if (l >= lower) m += w.of(l);
      eq += l == cut;
    });
    m = warp_all(m, Add());
    eq = warp_all(eq, Add());
    if (lane == 0) {
      sm.mass[warp] = m;
      sm.ties[warp] = eq;
    }
  } else {
    stretch(min(end, warp * seg), min(end, warp * seg + seg), &sm.mass[warp], &sm.ties[warp]);
  }
  __syncthreads();
  if (warp == 0) {
    const u64 m = warp_all(lane < ST_WARPS ? sm.mass[lane] : 0, Add());
    const unsigned eq = warp_all(lane < ST_WARPS ? sm.ties[lane] : 0, Add());
    if (lane == 0) {
      sm.cta_mass = m;
      sm.cta_ties = eq;
    }
  }
  cl.sync();
  // a lane a CTA of the row; every warp does the same
  const Shared* const o = cl.map_shared_rank(&sm, lane < nc ? lane : 0);
  u64 m = lane < nc ? o->cta_mass : 0;
  const unsigned eq = lane < nc ? o->cta_ties : 0;
  unsigned tie = warp_before(eq, lane);  // members at the cut before
  if (cut_in && tie < ties) m += min(eq, ties - tie) * cut_w;
  u64 left = warp_before(m, lane);
  const u64 target = __umul64hi(fraction(), __shfl_sync(0xffffffffu, left + m, 31));
  const unsigned hit = __ballot_sync(0xffffffffu, target >= left && target < left + m);
  left = target - __shfl_sync(0xffffffffu, left, rank);  // what remains before the target within this CTA, if it is here
  tie = __shfl_sync(0xffffffffu, tie, rank);
  if (hit >> rank & 1) {
    if (whole > 0) {
      __syncthreads();
      stretch(min(end, warp * seg), min(end, warp * seg + seg), &sm.mass[warp], &sm.ties[warp]);
      __syncthreads();
    }
    auto find = [&](const u64* mass, const unsigned* equal) {  // the part that holds the target; every warp does the same
      const unsigned eq = lane < ST_WARPS ? equal[lane] : 0, t = tie + warp_before(eq, lane);
      u64 v = lane < ST_WARPS ? mass[lane] : 0;
      if (cut_in && t < ties) v += min(eq, ties - t) * cut_w;
      const u64 run = warp_before(v, lane);
      const unsigned in = __ballot_sync(0xffffffffu, left >= run && left < run + v);
      const int k = in ? __ffs(in) - 1 : 0;
      left -= __shfl_sync(0xffffffffu, run, k);
      tie = __shfl_sync(0xffffffffu, t, k);
      return k;
    };
    const int j0 = min(end, find(sm.mass, sm.ties) * seg), j1 = min(end, j0 + seg), fine = ((seg + ST_WARPS - 1) / ST_WARPS + 31) / 32 * 32;
    stretch(min(j1, j0 + warp * fine), min(j1, j0 + warp * fine + fine), &sm.fine_mass[warp], &sm.fine_ties[warp]);
    __syncthreads();
    const int k = find(sm.fine_mass, sm.fine_ties);
    if (k == warp) {
      const int e = min(j1, j0 + k * fine + fine);
      for (int i0 = j0 + k * fine; i0 < e; i0 += 32) {
        const int j = i0 + lane;
        const float l = j < e ? slice[j] : CUDART_NAN_F;
        const unsigned eqs = __ballot_sync(0xffffffffu, l == cut);
        u64 v = l >= lower ? w.of(l) : 0;
        if (l == cut && cut_in && tie + __popc(eqs & ((1u << lane) - 1)) < ties) v = cut_w;
        tie += __popc(eqs);
        const u64 run = warp_before(v, lane) + v;
        const unsigned here = __ballot_sync(0xffffffffu, run > left);
        if (here) {
          if (lane == __ffs(here) - 1) a.out[row] = base + j - pad;
          break;
        }
        left -= __shfl_sync(0xffffffffu, run, 31);
      }
    }
  }
  cl.sync();  // no CTA leaves while another reads its shared memory
}

template <typename T>
void launch(const SampleArgs& a, cudaStream_t s) {
  // The smallest cluster whose slices still let three CTAs share an SM (64 rows of 50257: 18 us, 23 with slices half as long, 20 twice);
  // more CTAs a row while the batch leaves SMs idle.
  int nc = 1;
  while (nc < ST_MAX_CLUSTER && (a.vocab + nc - 1) / nc > 16384) nc *= 2;
  while (nc < ST_MAX_CLUSTER && (long long)a.rows * nc * 2 <= sm_count(current_device()) && a.vocab / nc > 2048) nc *= 2;
  const int per = (a.vocab + nc - 1) / nc;
  const int smem = (int)sizeof(Shared) + (per + 6) / 4 * 16;  // a slice and up to three places before it
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
