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
// go on over their keys.  The draw adds kept weights by warp, then by parts of the stretch that holds the target.
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
constexpr int ST_LIST = 64;                    // members of a step that a warp ranks
constexpr int ST_TABLE = 128;                  // 2^(i / 128)
constexpr double ST_ONE = 35184372088832.0;    // 2^45
constexpr double ST_OCTAVES = 46.0;            // further below the maximum weights are zero

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

struct alignas(16) Shared {
  double table[ST_TABLE];                      // ST_ONE 2^(i / 128)
  u64 part[2][ST_WARPS];                       // reductions by warp, used in turn
  u64 mass[ST_WARPS], fine_mass[ST_WARPS];     // draw: kept weight above the cut, by warp
  unsigned ties[ST_WARPS], fine_ties[ST_WARPS];  // draw: members at the cut, by warp
  unsigned lo[2][ST_BINS], hi[2][ST_BINS];     // histograms, used in turn: counts in lo, weights in both
  unsigned list[ST_LIST];                      // keys of a step's members (the first CTA's)
  int n_list;
  // what one thread finds for its CTA
  u64 found_mass;
  unsigned found_key, found_count;
  int found_bin;
};

// w of a logit l with steps_below(l) < ST_BINS - 1.  2^y = 2^(k / 128) e^r with k the nearest integer to 128 y and
// |r| <= ln 2 / 256, where the series to r^4 is off by 1e-15; adding 2^52 rounds to the integer that the low bits then hold.
struct Weigh {
  float m, per;                                // maximum; histogram steps per unit of the logit
  double m64, c;                               // 128 log2(e) / T
  const double* table;
  // steps below the maximum, monotone in l; 0 for the maximum itself, infinities included
  __device__ __forceinline__ float steps_below(float l) const { return l == m ? 0.f : fminf((m - l) * per, (float)(ST_BINS - 1)); }
  __device__ __forceinline__ u64 of(float l) const {
    const double z = ((double)l - m64) * c;
    const double magic = 6755399441055744.0;   // 1.5 * 2^52
    const double t = z + magic;
    const int k = __double2loint(t);
    const double f = z - (t - magic);
    constexpr double A = 0.0054152123481245727;  // ln 2 / 128
    const double q = f * (A + f * (A * A / 2 + f * (A * A * A / 6 + f * (A * A * A * A / 24))));
    const double two = table[k & (ST_TABLE - 1)];
    const double sc = __hiloint2double(__double2hiint(two) + ((k >> 7) << 20), __double2loint(two));
    const u64 w = (u64)__double_as_longlong(fma(sc, q, sc) + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52
    return l == m ? (u64)ST_ONE : w;
  }
  __device__ __forceinline__ u64 operator()(float l) const { return steps_below(l) < ST_BINS - 1 ? of(l) : 0; }
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
  v = 0;
  for (int k = threadIdx.x & 31; k < nc * ST_WARPS; k += 32) v = op(v, cl.map_shared_rank(&sm, k / ST_WARPS)->part[turn][k % ST_WARPS]);
  turn ^= 1;
  return warp_all(v, op);
}

// The CTA's logits to shared memory, cleaned; returns this thread's largest.  Rows may start anywhere: single values up to a
// 16-byte boundary, 16 bytes at a time from there on; `slice` is placed so that those land on 16 bytes too.
template <typename T>
__device__ __forceinline__ float load_slice(const T* x, float* slice, int n, int head) {
  constexpr int PER = 16 / sizeof(T);
  float top = -CUDART_INF_F;
  auto one = [&](int i) {
    const float l = clean(to_f(x[i]));
    slice[i] = l;
    top = fmaxf(top, l);
  };
  const int vecs = n > head ? (n - head) / PER : 0, tail = head + vecs * PER;
  if ((int)threadIdx.x < min(head, n)) one(threadIdx.x);
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
    for (int k = 0; k < PER; k += 4) *reinterpret_cast<float4*>(slice + head + i * PER + k) = make_float4(f[k], f[k + 1], f[k + 2], f[k + 3]);
  }
  if (n > head && tail + (int)threadIdx.x < n) one(tail + threadIdx.x);
  return top;
}

template <typename T>
__global__ void __launch_bounds__(ST_THREADS, 3) sample_tokens_kernel(SampleArgs a, int per) {
  extern __shared__ __align__(16) unsigned char dyn[];
  Shared& sm = *reinterpret_cast<Shared*>(dyn);
  cg::cluster_group cl = cg::this_cluster();
  const int nc = cl.num_blocks(), rank = cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / nc;
  const int base = rank * per, n = max(0, min(per, a.vocab - base));  // this CTA's logits
  if (tid < ST_TABLE) sm.table[tid] = exp2((double)tid / ST_TABLE) * ST_ONE;
  if (tid == 0) sm.n_list = 0;
  pdl_launch_dependents();
  pdl_wait();

  // ---- the row and its maximum
  const T* const x = (const T*)a.logits + row * a.ld + base;
  const int head = (int)((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T));
  float* const slice = reinterpret_cast<float*>(dyn + sizeof(Shared)) + (4 - head % 4) % 4;
  const float top = load_slice(x, slice, n, head);
  int turn = 0;
  const unsigned best = (unsigned)cluster_all(cl, nc, sm, top == -CUDART_INF_F ? 0 : key_of(top), turn, Larger());
  const double T_ = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
  Weigh w;
  w.m = of_key(best);
  if (best == 0 || !(T_ > 0.0)) {  // no possible token, or the most likely one: the lowest index that holds the maximum
    u64 first = 0;
    if (best != 0)
      for (int i = tid; i < n && !first; i += ST_THREADS)
        if (slice[i] == w.m) first = (unsigned)~(base + i);
    first = cluster_all(cl, nc, sm, first, turn, Larger());
    if (rank == 0 && tid == 0) a.out[row] = best == 0 ? -1 : (long long)(int)~(unsigned)first;
    cl.sync();  // no CTA leaves while another reads its shared memory
    return;
  }
  w.m64 = w.m;
  w.c = 1.4426950408889634074 / T_ * ST_TABLE;
  w.per = (float)(1.4426950408889634074 / T_ * ((ST_BINS - 1) / ST_OCTAVES));
  w.table = sm.table;
  const int top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
  const double top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
  const u64 min_w = (u64)ceil(fmax(0.0, fmin(a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p, 1.0)) * ST_ONE);
  const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.0;

  float cut = -CUDART_INF_F;  // kept: logits above the cut, and the first `ties` that equal it
  unsigned ties = 0;
  if (by_count || by_mass) {
    int h = 0;  // histogram in use
    auto clear = [&]() {
      sm.lo[h][tid] = sm.hi[h][tid] = 0;
      __syncthreads();
    };
    auto put = [&](int b, u64 v) {
      const unsigned low = (unsigned)v, old = atomicAdd(&sm.lo[h][b], low);
      const unsigned high = (unsigned)(v >> 32) + (old + low < old);
      if (high) atomicAdd(&sm.hi[h][b], high);
    };
    // The first bin at which the running sum over the cluster's histograms reaches `want`, -1: none.  The sum before it is added to
    // `before`.  Switches to the other histogram: this one is written again a cluster barrier after all have read it.
    auto crossing = [&](bool mass, u64 want, u64& before) {
      u64 v = 0;
#pragma unroll
      for (int r = 0; r < ST_MAX_CLUSTER; ++r) {
        if (r >= nc) break;
        const Shared* const o = cl.map_shared_rank(&sm, r);
        v += o->lo[h][tid];
        if (mass) v += (u64)o->hi[h][tid] << 32;
      }
      u64 run = warp_before(v, lane);
      if (lane == 31) sm.mass[warp] = run + v;
      if (tid == 0) sm.found_bin = -1;
      __syncthreads();
      run += before;
      for (int k = 0; k < warp; ++k) run += sm.mass[k];
      if (run < want && run + v >= want) {
        sm.found_bin = tid;
        sm.found_mass = run;
      }
      __syncthreads();
      const int bin = sm.found_bin;
      if (bin >= 0) before = sm.found_mass;
      h ^= 1;
      __syncthreads();
      return bin;
    };
    // The logit at which the sum reaches `want`, a member of step `bin` of the first histogram; `before` becomes the sum over
    // larger logits.
    auto narrow = [&](bool mass, u64 want, int bin, u64& before) {
      auto sub_step = [&](float l) {  // -1: not a member
        const float t = w.steps_below(l);
        return (int)t == bin ? (int)((t - bin) * ST_BINS) : -1;
      };
      clear();
#pragma unroll 4
      for (int i = tid; i < n; i += ST_THREADS) {
        const float l = slice[i];
        const int s = sub_step(l);
        if (s < 0) continue;
        if (mass) put(s, w.of(l));
        else atomicAdd(&sm.lo[h][s], 1u);
      }
      cl.sync();
      const int sub = crossing(mass, want, before);
      Shared* const first = cl.map_shared_rank(&sm, 0);
#pragma unroll 4
      for (int i = tid; i < n; i += ST_THREADS) {
        const float l = slice[i];
        if (sub_step(l) != sub) continue;
        const int k = atomicAdd(&first->n_list, 1);
        if (k < ST_LIST) first->list[k] = key_of(l);
      }
      cl.sync();
      const int members = first->n_list;
      if (members <= ST_LIST) {
        if (warp == 0) {
          // a lane weighs up to two members against all
          unsigned k[2];
          u64 v[2], over[2] = {before, before}, eq[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            k[e] = lane + 32 * e < members ? first->list[lane + 32 * e] : 0;
            v[e] = k[e] == 0 ? 0 : mass ? w(of_key(k[e])) : 1;
          }
          for (int j = 0; j < members; ++j) {
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
        const unsigned key = sm.found_key;
        cl.sync();  // the list may be filled again
        if (rank == 0 && tid == 0) sm.n_list = 0;
        cl.sync();
        return of_key(key);
      }
      // Many members in so narrow a step are equal ones, or nearly so.  Histograms over their keys, whose bounds are the bin's,
      // a hundredth of a bin wider than rounding could move them.
      const double high = (double)w.m - (bin - 0.01) / (double)w.per, low = (double)w.m - (bin + 1.01) / (double)w.per;
      unsigned k_hi = best, k_lo = key_of(clean(__double2float_rd(low)));
      if (bin > 0) k_hi = min(k_hi, key_of(clean(__double2float_ru(high))));
      while (true) {
        int shift = 0;
        while (((k_hi - k_lo) >> shift) >= ST_BINS) ++shift;
        clear();
        for (int i = tid; i < n; i += ST_THREADS) {
          const float l = slice[i];
          const unsigned k = key_of(l);
          if (k >= k_lo && k <= k_hi && sub_step(l) == sub) {
            if (mass) put((k_hi - k) >> shift, w.of(l));
            else atomicAdd(&sm.lo[h][(k_hi - k) >> shift], 1u);
          }
        }
        cl.sync();
        if (rank == 0 && tid == 0) sm.n_list = 0;
        const int s = crossing(mass, want, before);
        k_hi -= (unsigned)max(s, 0) << shift;  // a sum that reaches `want` among these members does so in one of their steps
        if (shift == 0) break;
        k_lo = max(k_lo, k_hi - ((1u << shift) - 1));
      }
      cl.sync();
      return of_key(k_hi);
    };

    // Without top_k, weights below (1 - top_p) / (2 vocab) cannot be where top_p is reached: all of them together weigh less than the rest.
    const u64 floor_w = by_count || !(top_p > 0.0) ? 0 : (u64)((1.0 - top_p) / a.vocab * (0.5 * ST_ONE));
    u64 total = 0, before = 0;
    bool counted = false;
    if (by_count) {
      clear();
#pragma unroll 4
      for (int i = tid; i < n; i += ST_THREADS) {
        const int b = (int)w.steps_below(slice[i]);
        if (b < ST_BINS - 1) atomicAdd(&sm.lo[h][b], 1u);
      }
      cl.sync();
      const int bin = crossing(false, (u64)top_k, before);
      if (bin >= 0) {  // else every possible token is among the first top_k
        cut = narrow(false, (u64)top_k, bin, before);
        ties = (unsigned)((u64)top_k - before);
        counted = true;
      }
    }
    if (by_mass) {
      clear();
#pragma unroll 2
      for (int i = tid; i < n; i += ST_THREADS) {
        const float l = slice[i];
        const float t = w.steps_below(l);
        if (t >= ST_BINS - 1 || l < cut) continue;
        const u64 v = w.of(l);
        if (l > cut) total += v;
        if (v > floor_w) put((int)t, v);
      }
      total = cluster_all(cl, nc, sm, total, turn, Add());
      if (counted) total += ties * w(cut);
      const double part = ceil((top_p > 0.0 ? top_p : 0.0) * (double)total);
      const u64 want = part >= 1.0 ? (part < (double)total ? (u64)part : total) : 1;
      before = 0;
      const int bin = crossing(true, want, before);
      if (bin >= 0) {  // else every token above the cut is needed
        const float at = narrow(true, want, bin, before);
        const u64 v = w(at);
        const unsigned some = (unsigned)((want - before + v - 1) / v);
        if (at > cut || some < ties) {
          cut = at;
          ties = some;
        }
      }
    }
  }

  // ---- draw.  A warp's stretch is contiguous; the one that holds the target is cut into a part for each warp of its CTA, and the
  // part that holds it is walked.
  const u64 cut_w = ties ? w(cut) : 0;
  const bool cut_in = cut_w != 0 && cut_w >= min_w;
  auto over_cut = [&](float l) -> u64 {  // weight of a logit above the cut, 0 where min_p takes it out
    if (!(l > cut) || !(w.steps_below(l) < ST_BINS - 1)) return 0;
    const u64 v = w.of(l);
    return v >= min_w ? v : 0;
  };
  auto stretch = [&](int s0, int s1, u64* mass, unsigned* equal) {
    u64 m = 0;
    unsigned eq = 0;
#pragma unroll 4
    for (int i = s0 + lane; i < s1; i += 32) {
      const float l = slice[i];
      m += over_cut(l);
      eq += l == cut;
    }
    m = warp_all(m, Add());
    eq = warp_all(eq, Add());
    if (lane == 0) {
      *mass = m;
      *equal = eq;
    }
  };
  const int seg = (per + ST_THREADS - 1) / ST_THREADS * 32;
  stretch(min(n, warp * seg), min(n, warp * seg + seg), &sm.mass[warp], &sm.ties[warp]);
  cl.sync();
  double u = a.uniform_f64 ? ((const double*)a.uniform)[row] : (double)((const float*)a.uniform)[row];
  u = u > 0.0 ? u : 0.0;
  int mine = -1;       // the target's stretch, where it is this CTA's
  u64 left = 0;        // target minus the kept weight before it
  unsigned tie = 0;    // members at the cut before it
  {
    // all stretches of the row in order, three a lane; every warp does the same
    constexpr int PER = (ST_MAX_CLUSTER * ST_WARPS + 31) / 32;
    u64 m[PER], all = 0;
    unsigned t[PER], sum_t = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int k = lane * PER + e;
      const bool there = k < nc * ST_WARPS;
      const Shared* const o = cl.map_shared_rank(&sm, there ? k / ST_WARPS : 0);
      m[e] = there ? o->mass[k % ST_WARPS] : 0;
      t[e] = there ? o->ties[k % ST_WARPS] : 0;
      sum_t += t[e];
    }
    unsigned run_t = warp_before(sum_t, lane);
    unsigned before_t[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      before_t[e] = run_t;
      if (cut_in && run_t < ties) m[e] += min(t[e], ties - run_t) * cut_w;
      run_t += t[e];
      all += m[e];
    }
    u64 run = warp_before(all, lane);
    const u64 sum = __shfl_sync(0xffffffffu, run + all, 31);
    const u64 target = __umul64hi(u < 1.0 ? (u64)(u * 18446744073709551616.0) : ~0ull, sum);
    int hit = -1;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (target >= run && target < run + m[e]) {
        hit = lane * PER + e;
        left = target - run;
        tie = before_t[e];
      }
      run += m[e];
    }
    const int from = __ffs(__ballot_sync(0xffffffffu, hit >= 0)) - 1;
    hit = __shfl_sync(0xffffffffu, hit, from);
    left = __shfl_sync(0xffffffffu, left, from);
    tie = __shfl_sync(0xffffffffu, tie, from);
    if (hit / ST_WARPS == rank) mine = hit % ST_WARPS;
  }
  if (mine >= 0) {
    const int s0 = min(n, mine * seg), s1 = min(n, s0 + seg), fine = (seg + ST_THREADS - 1) / ST_THREADS * 32;
    stretch(min(s1, s0 + warp * fine), min(s1, s0 + warp * fine + fine), &sm.fine_mass[warp], &sm.fine_ties[warp]);
    __syncthreads();
    int part = 0;
    for (; part < ST_WARPS - 1; ++part) {
      const u64 m = sm.fine_mass[part] + (cut_in && tie < ties ? min(sm.fine_ties[part], ties - tie) * cut_w : 0);
      if (left < m) break;
      left -= m;
      tie += sm.fine_ties[part];
    }
    if (part == warp) {
      const int e = min(s1, s0 + part * fine + fine);
      for (int i0 = s0 + part * fine; i0 < e; i0 += 32) {
        const int i = i0 + lane;
        const float l = i < e ? slice[i] : CUDART_NAN_F;
        const unsigned eqs = __ballot_sync(0xffffffffu, l == cut);
        u64 v = over_cut(l);
        if (l == cut && cut_in && tie + __popc(eqs & ((1u << lane) - 1)) < ties) v = cut_w;
        tie += __popc(eqs);
        const u64 run = warp_before(v, lane) + v;
        const unsigned hit = __ballot_sync(0xffffffffu, run > left);
        if (hit) {
          if (lane == __ffs(hit) - 1) a.out[row] = base + i;
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
  // Smallest cluster whose slices let three CTAs share an SM; more CTAs a row while the batch leaves SMs idle.
  int nc = 1;
  while (nc < ST_MAX_CLUSTER && (a.vocab + nc - 1) / nc > 8192) nc *= 2;
  while (nc < ST_MAX_CLUSTER && (long long)a.rows * nc * 2 <= sm_count(current_device()) && a.vocab / nc > 2048) nc *= 2;
  const int per = (a.vocab + nc - 1) / nc;
  const int smem = (int)sizeof(Shared) + per * 4 + 16;
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
