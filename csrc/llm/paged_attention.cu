// Attention of new tokens over a paged key / value cache:
//
//   s_j = f(scale q . K_j),  f(x) = x  or  softcap tanh(x / softcap)
//   out = sum_j exp(s_j - m) V_j / sum_j exp(s_j - m),  j in [max(0, kv_len - window), kv_len),  m = max s_j
//
// A token that sees no position gets zeros.  Every visible key and value is read once per (token, kv head): the cache's
// bytes are the bound (4 D bytes for 4 D H / Hkv operations), so the kernel is built around keeping loads in flight.
//
// Work: a (token, kv head, 16 of its query heads) is an item, its visible positions are cut into units of 64 keys.  The
// units of all items, in order, are dealt to a fixed grid in equal contiguous shares, from the lengths on the device:
// ragged batches stay balanced, one long sequence uses the whole GPU, and a captured launch fits every later length.  An item
// that lies in one share is finished there; one that was cut leaves (max, sum, output) parts, and whichever CTA arrives
// last at its counter joins them in share order, so the result does not depend on timing.
//
// Inside a CTA each of four warps owns 16 keys of a unit and its own ring of cp.async stages, without block barriers
// between units; the ring runs on across items.  Scores and outputs are m16n8k16 products with the item's query heads as
// the 16 rows (decode has too few rows for the 128-row tcgen05 tiles, and the tensor time here is a fraction of the load time).
// Maximum, sum and output are kept in 32 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "../api.h"
#include "../common/launch.h"
#include "../common/ptx.cuh"

namespace rt {

namespace {

constexpr int PA_WARPS = 4;
constexpr int PA_TILE = 16;                    // keys of one warp step, and query heads of an item
constexpr int PA_UNIT = PA_WARPS * PA_TILE;    // keys of one CTA step
constexpr float PA_LOG2E = 1.4426950408889634f;

template <typename T, int DP> struct Cfg {
  static constexpr int ROW = DP * 2 + 16;                      // bytes of a staged row: 16 more than the data keep ldmatrix conflict-free
  static constexpr int STAGES = DP <= 96 ? 3 : 2;
  static constexpr int STAGE = 2 * PA_TILE * ROW;              // one warp's K and V rows
  static constexpr int QBUF = PA_TILE * ROW;
  static constexpr int ACC_LD = DP + 8;                        // floats of a row of the merge buffer
  static constexpr int OFF_Q = STAGES * PA_WARPS * STAGE;
  static constexpr int OFF_ACC = OFF_Q + (STAGES + 1) * QBUF;
  static constexpr int OFF_ML = OFF_ACC + 2 * PA_TILE * ACC_LD * 4;
  static constexpr int OFF_TOK = OFF_ML + 2 * PA_WARPS * PA_TILE * 4;
  static constexpr int SMEM = OFF_TOK + PAGED_ATTN_CHUNK * 20 + 8;
  static constexpr bool Q_IN_REGS = DP <= 128;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool full) {  // zero-fills where not full
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_2x16<std::is_same<T, __half>::value>(lo, hi); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// What a chunk of tokens looks like to the schedule, in shared memory.
struct Tokens {
  long long* first;  // units of the tokens before this one, all heads
  int *lo, *len, *seq;
};

__device__ __forceinline__ int units_of(int lo, int len) { return (int)(((unsigned)(len - lo) + PA_UNIT - 1) / PA_UNIT); }

// A walk over the units of this CTA's share.
struct Walk {
  int t, hr;       // token; kv head * row tiles + row tile
  int v, nu;       // unit within the item, units of the item
};

template <typename T, int DP>
__global__ void __launch_bounds__(PA_WARPS * 32)
paged_attention_kernel(PagedAttnArgs a, int t0, int n, float* __restrict__ part, int* __restrict__ counters, int* __restrict__ status) {
  using C = Cfg<T, DP>;
  constexpr int S = C::STAGES, CH = DP / 8, NT = DP / 8, KS = DP / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ long long sm_scan[PA_WARPS];
  __shared__ int sm_mask[PA_WARPS][S];
  __shared__ int sm_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedCache& c = a.cache;
  const int G = a.H / c.Hkv, RT = (G + PA_TILE - 1) / PA_TILE, HR = c.Hkv * RT;
  const int chunks = c.D >> 3;
  Tokens tk;
  tk.first = reinterpret_cast<long long*>(smem + C::OFF_TOK);
  tk.lo = reinterpret_cast<int*>(tk.first + PAGED_ATTN_CHUNK + 1);
  tk.len = tk.lo + PAGED_ATTN_CHUNK;
  tk.seq = tk.len + PAGED_ATTN_CHUNK;
  if (c.D != DP) {  // columns that no copy fills
    for (int i = tid; i < C::OFF_ACC / 16; i += blockDim.x) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  }
  pdl_launch_dependents();
  pdl_wait();

  // ---- schedule: units of every token, summed
  constexpr int PER = PAGED_ATTN_CHUNK / (PA_WARPS * 32);
  const int per = (n + PA_WARPS * 32 - 1) / (PA_WARPS * 32);
  long long units[PER], mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = tid * per + i;
    units[i] = 0;
    if (i < per && t < n) {
      const int s = a.seq ? __ldcg(a.seq + t0 + t) : t0 + t;
      int len = __ldcg(a.kv_len + t0 + t);
      if (s == -1) len = 0;
      else if (s < 0 || s >= c.n_seq || len < 0 || len > (long long)c.max_pages * c.page) {
        if (blockIdx.x == 0) atomicCAS(status, 0, RT_ERR_BOUNDS);
        len = 0;
      }
      const int lo = a.window > 0 && len > a.window ? len - a.window : 0;
      tk.lo[t] = lo;
      tk.len[t] = len;
      tk.seq[t] = s;
      units[i] = (long long)units_of(lo, len) * HR;
    }
    mine += units[i];
  }
  long long run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) sm_scan[warp] = run;
  __syncthreads();
  long long U = 0, before = run - mine;
#pragma unroll
  for (int w = 0; w < PA_WARPS; ++w) {
    if (w < warp) before += sm_scan[w];
    U += sm_scan[w];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = tid * per + i;
    if (i < per && t < n) tk.first[t] = before;
    before += units[i];
  }
  if (tid == 0) tk.first[n] = U;
  __syncthreads();
  const int P = (int)min((long long)gridDim.x, U);  // every share holds a unit at least
  for (int t = blockIdx.x; t < n; t += gridDim.x)
    if (tk.len[t] == 0)
      for (int i = tid; i < a.H * c.D; i += blockDim.x) put((T*)a.out + (t0 + t) * a.o_st + (i / c.D) * a.o_sh + i % c.D, 0.f);
  if (blockIdx.x >= P) return;
  const long long ub = U * blockIdx.x / P, ue = U * (blockIdx.x + 1) / P;

  auto enter = [&](Walk& w, long long rem) {  // rem: units from the token's first
    w.nu = units_of(tk.lo[w.t], tk.len[w.t]);
    w.hr = (int)(rem / w.nu);
    w.v = (int)(rem % w.nu);
  };
  auto step = [&](Walk& w) {
    if (++w.v < w.nu) return;
    w.v = 0;
    if (++w.hr < HR) return;
    w.hr = 0;
    do ++w.t; while (w.t < n && tk.len[w.t] == 0);
    if (w.t < n) w.nu = units_of(tk.lo[w.t], tk.len[w.t]);
  };
  Walk ld;
  {
    int x = 0, y = n;  // last token whose first unit is <= ub
    while (y - x > 1) {
      const int mid = (x + y) >> 1;
      if (tk.first[mid] <= ub) x = mid;
      else y = mid;
    }
    ld.t = x;
    enter(ld, ub - tk.first[x]);
  }
  Walk cw = ld;

  // ---- loads: lane r < 16 looks up the page of the tile's key r one tile ahead
  const uint32_t sbase = smem_u32(smem);
  const uint32_t my_stage = sbase + warp * C::STAGE;
  long long lu = ub;
  int ld_items = 0;
  bool ld_new = true;
  int pg = -1, row_in_page = 0;
  auto look_up = [&]() {
    pg = -1;
    if (lu < ue && lane < PA_TILE) {
      const unsigned j = (unsigned)tk.lo[ld.t] + (unsigned)ld.v * PA_UNIT + warp * PA_TILE + lane;
      if (j < (unsigned)tk.len[ld.t]) {
        const unsigned k = j / (unsigned)c.page;
        row_in_page = (int)(j - k * c.page);
        pg = __ldcg(c.table + tk.seq[ld.t] * c.table_stride + k);
        if (pg < 0 || pg >= c.n_pages) {
          pg = -1;
          atomicCAS(status, 0, RT_ERR_BOUNDS);
        }
      }
    }
  };
  auto issue = [&](int stage) {
    if (lu < ue) {
      const unsigned mask = __ballot_sync(0xffffffffu, pg >= 0);
      if (lane == 0) sm_mask[warp][stage] = (int)mask;
      const int hk = ld.hr / RT;
      if (ld_new) {  // this warp's four rows of the item's queries
        const int r0 = (ld.hr - hk * RT) * PA_TILE;
        const uint32_t qd = sbase + C::OFF_Q + (ld_items % (S + 1)) * C::QBUF;
#pragma unroll
        for (int i = lane; i < 4 * CH; i += 32) {
          const int r = warp * 4 + i / CH, ch = i % CH;
          const bool ok = r0 + r < G;
          if (ch < chunks)
            cp_async16(qd + r * C::ROW + ch * 16, (const T*)a.q + (ok ? (t0 + ld.t) * a.q_st + (long long)(hk * G + r0 + r) * a.q_sh : 0) + ch * 8, ok);
        }
        ++ld_items;
      }
      if (mask) {
        const long long off = (long long)(pg < 0 ? 0 : pg) * c.s_page + (long long)row_in_page * c.s_row + (long long)hk * c.s_head;
        const uint32_t dst = my_stage + stage * (PA_WARPS * C::STAGE);
#pragma unroll
        for (int i = 0; i < PA_TILE * CH / 32; ++i) {
          const int r = (i * 32 + lane) / CH, ch = (i * 32 + lane) % CH;
          const long long o = __shfl_sync(0xffffffffu, off, r);
          const bool ok = mask >> r & 1;
          if (ch < chunks) {
            cp_async16(dst + r * C::ROW + ch * 16, ok ? (const T*)c.k + o + ch * 8 : (const T*)a.q, ok);
            cp_async16(dst + PA_TILE * C::ROW + r * C::ROW + ch * 16, ok ? (const T*)c.v + o + ch * 8 : (const T*)a.q, ok);
          }
        }
      }
      const int t_was = ld.t, h_was = ld.hr;
      ++lu;
      step(ld);
      ld_new = ld.t != t_was || ld.hr != h_was;
      look_up();
    }
    cp_commit();
  };
  __syncthreads();  // the zeroed columns are in place
  look_up();
#pragma unroll
  for (int i = 0; i < S; ++i) issue(i);

  // ---- items
  const float scale2 = a.softcap > 0.f ? a.scale / a.softcap * (2.f * PA_LOG2E) : a.scale * PA_LOG2E;
  const float cap2 = a.softcap * PA_LOG2E;
  float* acc_buf = reinterpret_cast<float*>(smem + C::OFF_ACC);
  float* sm_m = reinterpret_cast<float*>(smem + C::OFF_ML);
  float* sm_l = sm_m + PA_WARPS * PA_TILE;
  const uint32_t k_lane = ((lane >> 4) * 8 + (lane & 7)) * C::ROW + ((lane >> 3) & 1) * 16;
  const uint32_t v_lane = (((lane >> 3) & 1) * 8 + (lane & 7)) * C::ROW + (lane >> 4) * 16;
  int stage = 0, item = 0;
  long long u = ub;
  while (u < ue) {
    const int t = cw.t, hk = cw.hr / RT, r0 = (cw.hr - hk * RT) * PA_TILE, rows = min(PA_TILE, G - r0);
    const long long g0 = tk.first[t] + (long long)cw.hr * cw.nu, g1 = g0 + cw.nu;
    const long long end = min(g1, ue);
    uint32_t qf[C::Q_IN_REGS ? KS : 1][4];
    float o[NT][4], m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    cp_wait<S - 1>();
    __syncthreads();  // all four warps' query rows have arrived; the merge buffer is free again
    // ldmatrix A fragments: rows 0-7 / 8-15, columns 0-7 / 8-15 of each 16 x 16 block
    const uint32_t q_lane = sbase + C::OFF_Q + (item % (S + 1)) * C::QBUF + ((lane & 7) + ((lane >> 3) & 1) * 8) * C::ROW + (lane >> 4) * 16;
    if constexpr (C::Q_IN_REGS) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) ldsm4(q_lane + ks * 32, qf[ks]);
    }
    for (; u < end; ++u) {
      cp_wait<S - 1>();
      __syncwarp();
      const unsigned mask = (unsigned)sm_mask[warp][stage];
      if (mask) {
        const uint32_t ks_base = my_stage + stage * (PA_WARPS * C::STAGE);
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t b[4];
          ldsm4(ks_base + k_lane + ks * 32, b);
          if constexpr (C::Q_IN_REGS) {
            mma16816<T>(s0, qf[ks], b[0], b[1]);
            mma16816<T>(s1, qf[ks], b[2], b[3]);
          } else {
            uint32_t q4[4];
            ldsm4(q_lane + ks * 32, q4);
            mma16816<T>(s0, q4, b[0], b[1]);
            mma16816<T>(s1, q4, b[2], b[3]);
          }
        }
        // thread: rows lane / 4 (elements 0, 1) and lane / 4 + 8 (2, 3); keys 2 (lane % 4) + {0, 1}, and 8 more in s1
        const unsigned mk = mask >> (2 * (lane & 3));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s0[e] *= scale2;
          s1[e] *= scale2;
          if (a.softcap > 0.f) {  // tanh(x) = 1 - 2 / (exp(2x) + 1): its error is absolute, which is what a score's exponential sees
            s0[e] = cap2 - 2.f * cap2 / (ex2_approx(s0[e]) + 1.f);
            s1[e] = cap2 - 2.f * cap2 / (ex2_approx(s1[e]) + 1.f);
          }
          if (!(mk >> (e & 1) & 1)) s0[e] = -CUDART_INF_F;
          if (!(mk >> (8 + (e & 1)) & 1)) s1[e] = -CUDART_INF_F;
        }
        float x0 = fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s1[0], s1[1])), x1 = fmaxf(fmaxf(s0[2], s0[3]), fmaxf(s1[2], s1[3]));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
        if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
          const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
          const float f0 = n0 == -CUDART_INF_F ? 1.f : ex2_approx(m0 - n0), f1 = n1 == -CUDART_INF_F ? 1.f : ex2_approx(m1 - n1);
          m0 = n0;
          m1 = n1;
          l0 *= f0;
          l1 *= f1;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            o[i][0] *= f0;
            o[i][1] *= f0;
            o[i][2] *= f1;
            o[i][3] *= f1;
          }
        }
        const float b0 = m0 == -CUDART_INF_F ? 0.f : m0, b1 = m1 == -CUDART_INF_F ? 0.f : m1;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s0[e] = ex2_approx(s0[e] - b0);
          s1[e] = ex2_approx(s1[e] - b0);
          s0[2 + e] = ex2_approx(s0[2 + e] - b1);
          s1[2 + e] = ex2_approx(s1[2 + e] - b1);
        }
        l0 += (s0[0] + s0[1]) + (s1[0] + s1[1]);
        l1 += (s0[2] + s0[3]) + (s1[2] + s1[3]);
        const uint32_t p[4] = {pack2<T>(s0[0], s0[1]), pack2<T>(s0[2], s0[3]), pack2<T>(s1[0], s1[1]), pack2<T>(s1[2], s1[3])};
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
          uint32_t b[4];
          ldsm4_t(ks_base + PA_TILE * C::ROW + v_lane + i * 16, b);
          mma16816<T>(o[i], p, b[0], b[1]);
          mma16816<T>(o[i + 1], p, b[2], b[3]);
        }
      }
      __syncwarp();  // the stage is free
      issue(stage);
      stage = stage + 1 == S ? 0 : stage + 1;
      step(cw);
    }
    ++item;

    // ---- the four warps' states become one: warps 2, 3 hand over to 0, 1, whose sums all threads then add
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const int ra = lane >> 2, rb = ra + 8;
    if ((lane & 3) == 0) {
      sm_m[warp * PA_TILE + ra] = m0;
      sm_m[warp * PA_TILE + rb] = m1;
      sm_l[warp * PA_TILE + ra] = l0;
      sm_l[warp * PA_TILE + rb] = l1;
    }
    float* const buf = acc_buf + (warp & 1) * PA_TILE * C::ACC_LD + (lane & 3) * 2;
    if (warp >= 2) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (ra < rows) *reinterpret_cast<float2*>(buf + ra * C::ACC_LD + i * 8) = make_float2(o[i][0], o[i][1]);
        if (rb < rows) *reinterpret_cast<float2*>(buf + rb * C::ACC_LD + i * 8) = make_float2(o[i][2], o[i][3]);
      }
    }
    __syncthreads();
    auto top = [&](int r) {
      float x = sm_m[r];
#pragma unroll
      for (int w = 1; w < PA_WARPS; ++w) x = fmaxf(x, sm_m[w * PA_TILE + r]);
      return x;
    };
    auto factor = [](float m, float big) { return big == -CUDART_INF_F ? 0.f : ex2_approx(m - big); };
    if (warp < 2) {
      const float ta = top(ra), tb = top(rb);
      const float fa = factor(m0, ta), fb = factor(m1, tb);
      const float ga = factor(sm_m[(warp + 2) * PA_TILE + ra], ta), gb = factor(sm_m[(warp + 2) * PA_TILE + rb], tb);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (ra < rows) {
          float2* p = reinterpret_cast<float2*>(buf + ra * C::ACC_LD + i * 8);
          *p = make_float2(fmaf(p->x, ga, o[i][0] * fa), fmaf(p->y, ga, o[i][1] * fa));
        }
        if (rb < rows) {
          float2* p = reinterpret_cast<float2*>(buf + rb * C::ACC_LD + i * 8);
          *p = make_float2(fmaf(p->x, gb, o[i][2] * fb), fmaf(p->y, gb, o[i][3] * fb));
        }
      }
    }
    __syncthreads();
    auto total = [&](int r, float big) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) x += sm_l[w * PA_TILE + r] * factor(sm_m[w * PA_TILE + r], big);
      return x;
    };
    T* const out = (T*)a.out + (t0 + t) * a.o_st + (long long)(hk * G + r0) * a.o_sh;
    const bool whole = g0 >= ub && g1 <= ue;
    constexpr int PART = PA_TILE * (DP + 2);  // floats of a part: rows, maxima, sums
    float* const slot = part + ((long long)blockIdx.x * 2 + (g0 >= ub ? 1 : 0)) * PART;
    for (int i = tid; i < rows * DP; i += PA_WARPS * 32) {
      const int r = i / DP, d = i % DP;
      const float x = acc_buf[r * C::ACC_LD + d] + acc_buf[(PA_TILE + r) * C::ACC_LD + d];
      if (whole) {
        const float l = total(r, top(r));
        if (d < c.D) put(out + r * a.o_sh + d, l == 0.f ? 0.f : x / l);
      } else {
        __stcg(slot + r * DP + d, x);
        if (d == 0) {
          const float big = top(r);
          __stcg(slot + PA_TILE * DP + r, big);
          __stcg(slot + PA_TILE * (DP + 1) + r, total(r, big));
        }
      }
    }
    if (!whole) {
      const int c0 = (int)(((g0 + 1) * P - 1) / U), c1 = (int)((g1 * P - 1) / U);
      __threadfence();
      __syncthreads();
      if (tid == 0) sm_last = atomicAdd(&counters[c0], 1) == c1 - c0;
      __syncthreads();
      if (sm_last) {
        __threadfence();
        auto from = [&](int k) { return part + ((long long)k * 2 + (k == c0 ? 1 : 0)) * PART; };
        for (int i = tid; i < rows * c.D; i += PA_WARPS * 32) {
          const int r = i / c.D, d = i % c.D;
          float big = -CUDART_INF_F, x = 0.f, l = 0.f;
          for (int k = c0; k <= c1; ++k) big = fmaxf(big, __ldcg(from(k) + PA_TILE * DP + r));
          for (int k = c0; k <= c1; ++k) {
            const float* p = from(k);
            const float f = factor(__ldcg(p + PA_TILE * DP + r), big);
            x = fmaf(__ldcg(p + r * DP + d), f, x);
            l = fmaf(__ldcg(p + PA_TILE * (DP + 1) + r), f, l);
          }
          put(out + r * a.o_sh + d, l == 0.f ? 0.f : x / l);
        }
        if (tid == 0) counters[c0] = 0;  // for the next launch that uses this workspace
      }
    }
  }
  cp_wait<0>();
}

int occupancy_of(const void* kern, int smem) {
  int n = 0;
  RT_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  RT_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, PA_WARPS * 32, smem));
  return n < 1 ? 1 : n;
}

template <typename T, int DP>
int ctas_per_sm(int device) {
  static int occ[64] = {0};
  if (!occ[device]) occ[device] = occupancy_of((const void*)paged_attention_kernel<T, DP>, Cfg<T, DP>::SMEM);
  return occ[device];
}

template <typename T, int DP>
struct Run {
  static void go(const PagedAttnArgs& a, int grid, void* workspace, cudaStream_t s) {
    int* counters = reinterpret_cast<int*>(workspace);
    float* part = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + PAGED_ATTN_COUNTER_BYTES);
    for (int t0 = 0; t0 < a.n_tok; t0 += PAGED_ATTN_CHUNK) {
      launch_pdl(paged_attention_kernel<T, DP>, dim3(grid), dim3(PA_WARPS * 32), Cfg<T, DP>::SMEM, s, a, t0,
                 a.n_tok - t0 < PAGED_ATTN_CHUNK ? a.n_tok - t0 : PAGED_ATTN_CHUNK, part, counters, status_word(current_device()));
      RT_LAUNCH_CHECK();
    }
  }
};

template <typename F> auto by_width(int D, F f) {
  if (D <= 32) return f(std::integral_constant<int, 32>());
  if (D <= 64) return f(std::integral_constant<int, 64>());
  if (D <= 96) return f(std::integral_constant<int, 96>());
  if (D <= 128) return f(std::integral_constant<int, 128>());
  if (D <= 192) return f(std::integral_constant<int, 192>());
  return f(std::integral_constant<int, 256>());
}

}  // namespace

PagedAttnPlan paged_attention_plan(const PagedAttnArgs& a) {
  const int dev = current_device();
  return by_width(a.cache.D, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    const int occ = a.dtype == DT_F16 ? ctas_per_sm<__half, DP>(dev) : ctas_per_sm<__nv_bfloat16, DP>(dev);
    // no more CTAs than the longest lengths the table allows could use
    const int G = a.H / a.cache.Hkv;
    long long longest = (long long)a.cache.max_pages * a.cache.page;
    if (a.window > 0 && longest > a.window) longest = a.window;
    const long long most = (long long)(a.n_tok < PAGED_ATTN_CHUNK ? a.n_tok : PAGED_ATTN_CHUNK) * a.cache.Hkv * ((G + PA_TILE - 1) / PA_TILE) *
                           ((longest + PA_UNIT - 1) / PA_UNIT);
    PagedAttnPlan p;
    p.grid = (int)std::max(1ll, std::min<long long>((long long)occ * sm_count(dev), most));
    p.workspace_bytes = PAGED_ATTN_COUNTER_BYTES + (long long)occ * sm_count(dev) * 2 * PA_TILE * (DP + 2) * 4;
    return p;
  });
}

void paged_attention(const PagedAttnArgs& a, const PagedAttnPlan& p, void* workspace, cudaStream_t s) {
  if (a.n_tok == 0) return;
  RT_CHECK(a.cache.D % 8 == 0 && a.cache.D <= 256 && p.grid * 4 <= PAGED_ATTN_COUNTER_BYTES, "paged_attention: unsupported sizes");
  by_width(a.cache.D, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    if (a.dtype == DT_F16) Run<__half, DP>::go(a, p.grid, workspace, s);
    else Run<__nv_bfloat16, DP>::go(a, p.grid, workspace, s);
    return 0;
  });
}

}  // namespace rt
