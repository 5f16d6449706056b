// Attention of new tokens over a paged key / value cache:
//
//   s_j = f(scale q . K_j),  f(x) = x  or  softcap tanh(x / softcap)
//   out = sum_j exp(s_j - m) V_j / sum_j exp(s_j - m),  j in [max(0, kv_len - window), kv_len),  m = max s_j
//
// A token that sees no position gets zeros.  Every visible key and value is read once per (token, kv head): the cache's
// bytes are the bound (4 D bytes for 4 D H / Hkv operations), so the kernel is built around keeping loads in flight.
//
// Work: a (token, kv head, up to 8 or 16 of its query heads) is an item, its visible positions are cut into units of 64
// keys.  The units of all items, in order, are dealt to a fixed grid in equal contiguous shares, from the lengths on the
// device: ragged batches stay balanced, one long sequence uses the whole GPU, and a captured launch fits every later length.  An
// item that lies in one share is finished there; one that was cut leaves (max, sum, output) parts, and whichever CTA
// arrives last at its counter joins them in share order, so the result does not depend on timing.
//
// Inside a CTA each of four warps owns 16 keys of a unit and its own ring of cp.async stages, without block barriers
// between units; the ring runs on across items.  The products are m16n8k16 with the cache as the 16 rows and eight query
// heads as the columns: S^T = K Q^T (16 keys), O^T += V^T P^T (16 of D).  Decode has 1 to 16 query heads a kv head, a
// corner of a 128-row tcgen05 tile; here the tensor time is a fraction of the load time.  A lane copies parts of exactly
// the two key rows whose scores it later holds, so its page look-ups give its mask too.
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
constexpr int PA_TILE = 16;                    // keys of one warp step
constexpr int PA_UNIT = PA_WARPS * PA_TILE;    // keys of one CTA step
constexpr float PA_LOG2E = 1.4426950408889634f;
// The running maximum is moved only when a score exceeds it by PA_SLACK (base 2), and then set PA_ROOM below the score: weights
// reach 2^14 at most, which fits fp16, and small ones keep more of its digits than with the maximum itself.
constexpr float PA_SLACK = 14.f, PA_ROOM = 4.f;

template <int DP, int NH> struct Cfg {         // DP: head size rounded up, NH: eights of query heads in an item
  static constexpr int HEADS = 8 * NH;
  static constexpr int ROW = DP * 2 + 16;                      // bytes of a staged row: 16 more than the data keep ldmatrix conflict-free
  static constexpr int STAGES = DP <= 96 ? 3 : 2;
  static constexpr int STAGE = 2 * PA_TILE * ROW;              // one warp's K and V rows
  static constexpr int QBUF = HEADS * ROW;
  static constexpr int ACC_LD = DP + 4;                        // floats of a row of the merge buffer
  static constexpr int OFF_Q = STAGES * PA_WARPS * STAGE;
  static constexpr int OFF_ACC = OFF_Q + (STAGES + 1) * QBUF;
  static constexpr int OFF_ML = OFF_ACC + 2 * HEADS * ACC_LD * 4;
  static constexpr int OFF_TOK = OFF_ML + 2 * PA_WARPS * HEADS * 4;
  static constexpr int SMEM = OFF_TOK + PAGED_ATTN_CHUNK * 20 + 8;
  static constexpr int PART = HEADS * (DP + 2);                // floats of a part: rows, maxima, sums
  static constexpr bool Q_IN_REGS = DP * NH <= 256;
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
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {  // of 16-bit values across the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
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
  int t, hr;       // token; kv head * head groups + head group
  int v, nu;       // unit within the item, units of the item
};

template <typename T, int DP, int NH>
__global__ void __launch_bounds__(PA_WARPS * 32)
paged_attention_kernel(PagedAttnArgs a, unsigned page_mul, int page_shift, int t0, int n, float* __restrict__ part,
                       int* __restrict__ counters, int* __restrict__ status) {
  using C = Cfg<DP, NH>;
  constexpr int S = C::STAGES, CH = DP / 8, CL = CH / 4, KS = DP / 16, NT = DP / 16, HEADS = C::HEADS;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ long long sm_scan[PA_WARPS];
  __shared__ int sm_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedCache& c = a.cache;
  const int G = a.H / c.Hkv, RT = (G + HEADS - 1) / HEADS, HR = c.Hkv * RT;
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

  // ---- loads: lane copies 16-byte chunks lane % 4, + 4, .. of key rows lane / 4 and lane / 4 + 8; pages are looked up one tile ahead
  const uint32_t sbase = smem_u32(smem);
  const uint32_t my_stage = sbase + warp * C::STAGE + (lane >> 2) * C::ROW + (lane & 3) * 16;
  const T* const nothing = (const T*)a.q;  // source address of copies that only write zeros
  const int ch0 = lane & 3;
  const T* const kbase = (const T*)c.k + ch0 * 8;
  const T* const vbase = (const T*)c.v + ch0 * 8;
  long long left = ue - ub;                // units to load
  int ld_items = 0;
  bool ld_new = true;
  unsigned j0, jn;                         // this lane's first key of the next tile, the sequence's end
  const int* pages;
  long long head_off;
  auto enter_item = [&]() {
    jn = (unsigned)tk.len[ld.t];
    j0 = (unsigned)tk.lo[ld.t] + (unsigned)ld.v * PA_UNIT + warp * PA_TILE + (lane >> 2);
    pages = c.table + tk.seq[ld.t] * c.table_stride;
    head_off = (long long)(ld.hr / RT) * c.s_head;
  };
  int pg[2], row[2];
  auto look_up = [&]() {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const unsigned j = j0 + 8 * e;
      pg[e] = -1;
      if (j < jn) {
        const unsigned k = __umulhi(2 * j, page_mul) >> page_shift;  // j / page
        row[e] = (int)(j - k * c.page);
        pg[e] = __ldcg(pages + k);
        if (pg[e] < 0 || pg[e] >= c.n_pages) {
          pg[e] = -1;
          atomicCAS(status, 0, RT_ERR_BOUNDS);
        }
      }
    }
  };
  unsigned seen = 0;  // two bits a stage: whether this lane's two keys count
  auto issue = [&](int stage) {
    if (left > 0) {
      if (ld_new) {  // this warp's quarter of the item's query rows
        const int hk = ld.hr / RT, r0 = (ld.hr - hk * RT) * HEADS;
        const uint32_t qd = sbase + C::OFF_Q + (ld_items % (S + 1)) * C::QBUF;
#pragma unroll
        for (int i = lane; i < HEADS / 4 * CH; i += 32) {
          const int r = warp * (HEADS / 4) + i / CH, ch = i % CH;
          const bool ok = r0 + r < G;
          if (ch < chunks)
            cp_async16(qd + r * C::ROW + ch * 16, (const T*)a.q + (ok ? (t0 + ld.t) * a.q_st + (long long)(hk * G + r0 + r) * a.q_sh : 0) + ch * 8, ok);
        }
        ++ld_items;
      }
      const bool ok[2] = {pg[0] >= 0, pg[1] >= 0};
      seen = (seen & ~(3u << (2 * stage))) | ((ok[0] ? 1u : 0u) | (ok[1] ? 2u : 0u)) << (2 * stage);
      if (__any_sync(0xffffffffu, ok[0] || ok[1])) {
        const uint32_t dst = my_stage + stage * (PA_WARPS * C::STAGE);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const long long off = pg[e] * c.s_page + row[e] * c.s_row + head_off;
          const T* const ks = ok[e] ? kbase + off : nothing;
          const T* const vs = ok[e] ? vbase + off : nothing;
#pragma unroll
          for (int i = 0; i < CL; ++i)
            if (ch0 + 4 * i < chunks) {
              cp_async16(dst + e * 8 * C::ROW + i * 64, ok[e] ? ks + i * 32 : nothing, ok[e]);
              cp_async16(dst + (PA_TILE + e * 8) * C::ROW + i * 64, ok[e] ? vs + i * 32 : nothing, ok[e]);
            }
        }
      }
      --left;
      ld_new = ld.v + 1 == ld.nu;
      j0 += PA_UNIT;
      step(ld);
      pg[0] = pg[1] = -1;
      if (left > 0) {
        if (ld_new) enter_item();
        look_up();
      }
    }
    cp_commit();
  };
  __syncthreads();  // the zeroed columns are in place
  enter_item();
  look_up();
#pragma unroll
  for (int i = 0; i < S; ++i) issue(i);

  // ---- items
  const float scale2 = a.softcap > 0.f ? a.scale / a.softcap * (2.f * PA_LOG2E) : a.scale * PA_LOG2E;
  const float cap2 = a.softcap * PA_LOG2E;
  float* acc_buf = reinterpret_cast<float*>(smem + C::OFF_ACC);
  float* sm_m = reinterpret_cast<float*>(smem + C::OFF_ML);
  float* sm_l = sm_m + PA_WARPS * HEADS;
  // ldmatrix lanes: A fragments of K (rows are keys) and, transposed, of V; B fragments of Q
  const uint32_t k_lane = sbase + warp * C::STAGE + ((lane & 7) + ((lane >> 3) & 1) * 8) * C::ROW + (lane >> 4) * 16;
  const uint32_t v_lane = sbase + warp * C::STAGE + (PA_TILE + (lane & 7) + (lane >> 4) * 8) * C::ROW + ((lane >> 3) & 1) * 16;
  int stage = 0, item = 0;
  long long u = ub;
  while (u < ue) {
    const int t = cw.t, hk = cw.hr / RT, r0 = (cw.hr - hk * RT) * HEADS, rows = min(HEADS, G - r0);
    const long long g0 = tk.first[t] + (long long)cw.hr * cw.nu, g1 = g0 + cw.nu;
    const long long end = min(g1, ue);
    uint32_t qf[C::Q_IN_REGS ? NH : 1][C::Q_IN_REGS ? KS / 2 : 1][4];
    // this lane: heads 2 (lane % 4) + {0, 1} of each eight; rows (keys, or places in D) lane / 4 and lane / 4 + 8
    float o[NH][NT][4], m[NH][2], l[NH][2];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      m[h][0] = m[h][1] = -CUDART_INF_F;
      l[h][0] = l[h][1] = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[h][i][0] = o[h][i][1] = o[h][i][2] = o[h][i][3] = 0.f;
    }
    cp_wait<S - 1>();
    __syncthreads();  // all four warps' query rows have arrived; the merge buffer is free again
    const uint32_t q_lane = sbase + C::OFF_Q + (item % (S + 1)) * C::QBUF + (lane & 7) * C::ROW + (lane >> 3) * 16;
    if constexpr (C::Q_IN_REGS) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int k2 = 0; k2 < KS / 2; ++k2) ldsm4(q_lane + h * 8 * C::ROW + k2 * 64, qf[h][k2]);
    }
    for (; u < end; ++u) {
      cp_wait<S - 1>();
      __syncwarp();
      const bool ok0 = seen >> (2 * stage) & 1, ok1 = seen >> (2 * stage) & 2;
      if (__any_sync(0xffffffffu, ok0 || ok1)) {
        const uint32_t st = stage * (PA_WARPS * C::STAGE);
        float s[NH][2][4];  // even and odd steps of D, so that two chains of products run at once
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][0][e] = s[h][1][e] = 0.f;
#pragma unroll
        for (int k2 = 0; k2 < KS / 2; ++k2) {
          uint32_t ka[4], kb[4];
          ldsm4(k_lane + st + k2 * 64, ka);
          ldsm4(k_lane + st + k2 * 64 + 32, kb);
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            uint32_t q4[4];
            if constexpr (C::Q_IN_REGS) {
#pragma unroll
              for (int e = 0; e < 4; ++e) q4[e] = qf[h][k2][e];
            } else {
              ldsm4(q_lane + h * 8 * C::ROW + k2 * 64, q4);
            }
            mma16816<T>(s[h][0], ka, q4[0], q4[1]);
            mma16816<T>(s[h][1], kb, q4[2], q4[3]);
          }
        }
        bool grow = false;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = (s[h][0][e] + s[h][1][e]) * scale2;
            if (a.softcap > 0.f) x = cap2 - 2.f * cap2 / (ex2_approx(x) + 1.f);  // tanh(y) = 1 - 2 / (exp(2y) + 1), error absolute as a score's may be
            x = (e < 2 ? ok0 : ok1) ? x : -CUDART_INF_F;
            grow |= x > m[h][e & 1] + PA_SLACK;
            s[h][0][e] = x;
          }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = fmaxf(s[h][0][e], s[h][0][e + 2]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
              if (x > m[h][e] + PA_SLACK) {
                const float f = ex2_approx(m[h][e] - (x - PA_ROOM));
                m[h][e] = x - PA_ROOM;
                l[h][e] *= f;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                  o[h][i][e] *= f;
                  o[h][i][e + 2] *= f;
                }
              }
            }
        }
        uint32_t p[NH][2];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][0][e] = ex2_approx(s[h][0][e] - (m[h][e & 1] == -CUDART_INF_F ? 0.f : m[h][e & 1]));
          l[h][0] += s[h][0][0] + s[h][0][2];
          l[h][1] += s[h][0][1] + s[h][0][3];
          p[h][0] = transpose8x8(pack2<T>(s[h][0][0], s[h][0][1]));  // weights enter the product rounded to the values' type
          p[h][1] = transpose8x8(pack2<T>(s[h][0][2], s[h][0][3]));
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          uint32_t va[4];
          ldsm4_t(v_lane + st + i * 32, va);
#pragma unroll
          for (int h = 0; h < NH; ++h) mma16816<T>(o[h][i], va, p[h][0], p[h][1]);
        }
      }
      __syncwarp();  // the stage is free
      issue(stage);
      stage = stage + 1 == S ? 0 : stage + 1;
      step(cw);
    }
    ++item;

    // ---- the four warps' states become one: warps 2, 3 hand over to 0, 1, whose sums all threads then add
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], d);
        if (lane < 4) {
          sm_m[warp * HEADS + h * 8 + lane * 2 + e] = m[h][e];
          sm_l[warp * HEADS + h * 8 + lane * 2 + e] = l[h][e];
        }
      }
    float* const buf = acc_buf + (warp & 1) * HEADS * C::ACC_LD + (lane & 3) * 2 * C::ACC_LD + (lane >> 2);
    if (warp >= 2) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) buf[(h * 8 + (e & 1)) * C::ACC_LD + i * 16 + (e >> 1) * 8] = o[h][i][e];
    }
    __syncthreads();
    auto top = [&](int r) {
      float x = sm_m[r];
#pragma unroll
      for (int w = 1; w < PA_WARPS; ++w) x = fmaxf(x, sm_m[w * HEADS + r]);
      return x;
    };
    auto factor = [](float m, float big) { return big == -CUDART_INF_F ? 0.f : ex2_approx(m - big); };
    if (warp < 2) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        float f[2], g[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = h * 8 + (lane & 3) * 2 + e;
          const float big = top(r);
          f[e] = factor(m[h][e], big);
          g[e] = factor(sm_m[(warp + 2) * HEADS + r], big);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float* x = buf + (h * 8 + (e & 1)) * C::ACC_LD + i * 16 + (e >> 1) * 8;
            *x = fmaf(*x, g[e & 1], o[h][i][e] * f[e & 1]);
          }
      }
    }
    __syncthreads();
    auto total = [&](int r, float big) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) x += sm_l[w * HEADS + r] * factor(sm_m[w * HEADS + r], big);
      return x;
    };
    T* const out = (T*)a.out + (t0 + t) * a.o_st + (long long)(hk * G + r0) * a.o_sh;
    const bool whole = g0 >= ub && g1 <= ue;
    float* const slot = part + ((long long)blockIdx.x * 2 + (g0 >= ub ? 1 : 0)) * C::PART;
    for (int i = tid; i < rows * DP; i += PA_WARPS * 32) {
      const int r = i / DP, d = i % DP;
      const float x = acc_buf[r * C::ACC_LD + d] + acc_buf[(HEADS + r) * C::ACC_LD + d];
      if (whole) {
        const float l = total(r, top(r));
        if (d < c.D) put(out + r * a.o_sh + d, l == 0.f ? 0.f : x / l);
      } else {
        __stcg(slot + r * DP + d, x);
        if (d == 0) {
          const float big = top(r);
          __stcg(slot + HEADS * DP + r, big);
          __stcg(slot + HEADS * (DP + 1) + r, total(r, big));
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
        auto from = [&](int k) { return part + ((long long)k * 2 + (k == c0 ? 1 : 0)) * C::PART; };
        for (int i = tid; i < rows * c.D; i += PA_WARPS * 32) {
          const int r = i / c.D, d = i % c.D;
          float big = -CUDART_INF_F, x = 0.f, l = 0.f;
          for (int k = c0; k <= c1; ++k) big = fmaxf(big, __ldcg(from(k) + HEADS * DP + r));
          for (int k = c0; k <= c1; ++k) {
            const float* p = from(k);
            const float f = factor(__ldcg(p + HEADS * DP + r), big);
            x = fmaf(__ldcg(p + r * DP + d), f, x);
            l = fmaf(__ldcg(p + HEADS * (DP + 1) + r), f, l);
          }
          put(out + r * a.o_sh + d, l == 0.f ? 0.f : x / l);
        }
        if (tid == 0) counters[c0] = 0;  // for the next launch that uses this workspace
      }
    }
  }
  cp_wait<0>();
}

template <typename T, int DP, int NH>
int ctas_per_sm(int device) {
  static int occ[64] = {0};
  if (!occ[device]) {
    int n = 0;
    RT_CUDA_CHECK(cudaFuncSetAttribute((const void*)paged_attention_kernel<T, DP, NH>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DP, NH>::SMEM));
    RT_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, paged_attention_kernel<T, DP, NH>, PA_WARPS * 32, Cfg<DP, NH>::SMEM));
    RT_CHECK(n >= 1, "paged_attention: the kernel does not fit an SM");
    occ[device] = n;
  }
  return occ[device];
}

template <typename F, int DP> auto by_heads(const PagedAttnArgs& a, F f, std::integral_constant<int, DP> dp) {
  const bool one = a.H / a.cache.Hkv <= 8;
  if (a.dtype == DT_F16) return one ? f(__half(), dp, std::integral_constant<int, 1>()) : f(__half(), dp, std::integral_constant<int, 2>());
  return one ? f(__nv_bfloat16(), dp, std::integral_constant<int, 1>()) : f(__nv_bfloat16(), dp, std::integral_constant<int, 2>());
}
template <typename F> auto dispatch(const PagedAttnArgs& a, F f) {
  const int D = a.cache.D;
  if (D <= 32) return by_heads(a, f, std::integral_constant<int, 32>());
  if (D <= 64) return by_heads(a, f, std::integral_constant<int, 64>());
  if (D <= 96) return by_heads(a, f, std::integral_constant<int, 96>());
  if (D <= 128) return by_heads(a, f, std::integral_constant<int, 128>());
  if (D <= 192) return by_heads(a, f, std::integral_constant<int, 192>());
  return by_heads(a, f, std::integral_constant<int, 256>());
}

}  // namespace

PagedAttnPlan paged_attention_plan(const PagedAttnArgs& a) {
  const int dev = current_device();
  return dispatch(a, [&](auto type, auto dp, auto nh) {
    constexpr int DP = decltype(dp)::value, NH = decltype(nh)::value;
    const long long ctas = (long long)ctas_per_sm<decltype(type), DP, NH>(dev) * sm_count(dev);
    // no more CTAs than the longest lengths the table allows could use
    const int G = a.H / a.cache.Hkv;
    long long longest = (long long)a.cache.max_pages * a.cache.page;
    if (a.window > 0 && longest > a.window) longest = a.window;
    const long long most = (long long)std::min(a.n_tok, PAGED_ATTN_CHUNK) * a.cache.Hkv * ((G + 8 * NH - 1) / (8 * NH)) *
                           ((longest + PA_UNIT - 1) / PA_UNIT);
    PagedAttnPlan p;
    p.grid = (int)std::max(1ll, std::min(ctas, most));
    p.workspace_bytes = PAGED_ATTN_COUNTER_BYTES + ctas * 2 * Cfg<DP, NH>::PART * 4;
    return p;
  });
}

void paged_attention(const PagedAttnArgs& a, const PagedAttnPlan& p, void* workspace, cudaStream_t s) {
  if (a.n_tok == 0) return;
  RT_CHECK(a.cache.D % 8 == 0 && a.cache.D <= 256 && p.grid * 4 <= PAGED_ATTN_COUNTER_BYTES, "paged_attention: unsupported sizes");
  int* counters = reinterpret_cast<int*>(workspace);
  float* part = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + PAGED_ATTN_COUNTER_BYTES);
  int* status = status_word(current_device());
  // j / page for j < 2^31 as umulhi(2 j, mul) >> shift: with page <= 2^shift the product is off by less than j page / 2^(31 + shift) < 1
  int shift = 0;
  while ((1ll << shift) < a.cache.page) ++shift;
  const unsigned mul = (unsigned)((1ull << (31 + shift)) / (unsigned)a.cache.page + 1);
  dispatch(a, [&](auto type, auto dp, auto nh) {
    constexpr int DP = decltype(dp)::value, NH = decltype(nh)::value;
    for (int t0 = 0; t0 < a.n_tok; t0 += PAGED_ATTN_CHUNK) {
      launch_pdl(paged_attention_kernel<decltype(type), DP, NH>, dim3(p.grid), dim3(PA_WARPS * 32), Cfg<DP, NH>::SMEM, s, a, mul, shift, t0,
                 std::min(a.n_tok - t0, PAGED_ATTN_CHUNK), part, counters, status);
      RT_LAUNCH_CHECK();
    }
    return 0;
  });
}

}  // namespace rt
