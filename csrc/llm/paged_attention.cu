// Attention of new tokens over a paged key / value cache:
//
//   s_j = f(scale q . K_j),  f(x) = x  or  softcap tanh(x / softcap)
//   out = sum_j exp(s_j - m) V_j / sum_j exp(s_j - m),  j in [max(0, kv_len - window), kv_len),  m = max s_j
//
// A token that sees no position gets zeros.  Every visible key and value is read once per (token, kv head, 16 of its query heads): the
// cache's bytes are the bound (4 D bytes for 4 D H / Hkv operations), so the kernel is built around keeping loads in flight.
//
// Work: a (token, kv head, up to 8 or 16 of its query heads) is an item, its visible positions are cut into units of 64
// keys.  The units of all items, in order, are dealt to a fixed grid in equal contiguous shares, from the lengths on the
// device: ragged batches stay balanced, one long sequence uses the whole GPU, and a captured launch fits every later length.  An
// item that lies in one share is finished there; one that was cut leaves (max, sum, output) parts, and whichever CTA
// arrives last at its counter joins them in share order, so the result does not depend on timing.
//
// Inside a CTA each of four warps owns 16 keys of a unit and its own ring of stages, without block barriers between
// units; the ring runs on across items.  Rows are copied by cp.async with their 16-byte pieces on neighbouring lanes: 131072 keys
// (32 heads on 8, D = 128) take 94 to 97 us, 5.5 to 5.7 TB/s.  When they took 94, the same rows in 64-byte steps on four lanes
// took 122 us, as one bulk copy each 124 us (the copy engine takes one every 8 cycles, and a tile is 32 of them); keys and
// values as two groups, refilled one after the other, 118 us; a window of 32 block-table entries in registers 100 us.
// The products are m16n8k16 with the cache as the 16 rows and eight query heads as the columns: S^T = K Q^T (16 keys),
// O^T += V^T P^T (16 of D).  Decode has 1 to 16 query heads a kv head, a corner of a 128-row tcgen05 tile; here the tensor
// time is a fraction of the load time.  Weights enter the second product as two values of the cache's type, what fits the
// first and what that left, 16 bits together in bf16 and 22 in fp16: the result's own rounding is then the only one of its size
// (131072 keys take 96.9 us, 96.0 with weights rounded once; 64 sequences of 1 to 8192 keys in fp16 141 and 139).
// Rows that are not visible are not copied: a tile that has some masks their scores, and their values too, which may be left-over NaN.
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
// Units of a share at least: 4 sequences of 4000 keys on one head 37 us with one, 22 with two, 22 with four; 77 keys of 32 heads
// 9, 6.7, 9.5 us; 2048 keys of 8 heads 11.6, 11.2, 12.4.
constexpr int PA_MIN_SHARE = 2;
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
  static constexpr int OFF_FAC = OFF_ML + (2 * PA_WARPS + 3) * HEADS * 4;
  static constexpr int OFF_TOK = OFF_FAC + 32 * HEADS * 4;
  static constexpr int SMEM = OFF_TOK + PAGED_ATTN_CHUNK * 20 + 8;
  static constexpr int PART = HEADS * (DP + 2);                // floats of a part: rows, maxima, sums
  static constexpr bool Q_IN_REGS = DP * NH <= 256;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
// Two weights as sums of two values of type T, packed: the first is cut off strictly below the weight, so that the second is positive
// too and an infinite value times a weight stays infinite.  (fp16 cannot hold a second part below 2^-24: weights from 2^-10 on, of 2^4
// and more for the largest, get that.)
template <typename T> __device__ __forceinline__ void split2(float a, float b, uint32_t& first, uint32_t& second) {
  const uint32_t x = __float_as_uint(fmaxf(a, 1.17549435e-38f)) - 1, y = __float_as_uint(fmaxf(b, 1.17549435e-38f)) - 1;
  if constexpr (std::is_same<T, __half>::value) {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(first) : "f"(__uint_as_float(y)), "f"(__uint_as_float(x)));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&first));
    const float r = a - f.x, s = b - f.y;
    second = pack2<T>(a >= 0x1p-10f ? fmaxf(r, 0x1p-24f) : r, b >= 0x1p-10f ? fmaxf(s, 0x1p-24f) : s);
  } else {
    first = __byte_perm(x, y, 0x7632);
    second = pack2<T>(a - __uint_as_float(x & 0xffff0000u), b - __uint_as_float(y & 0xffff0000u));
  }
}
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// 1 - 2 / (exp(2x) + 1) is off by 2^-22 of one; near zero, where that would be much of the result, four terms of the series
// x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 (the next is below 2e-9 of x for |x| < 1/8).
__device__ __forceinline__ float tanh_of(float x) {
  const float q = x * x;
  const float near = x * fmaf(q, fmaf(q, fmaf(q, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  const float far = 1.f - 2.f / (ex2_approx(x * (2.f * PA_LOG2E)) + 1.f);
  return q < 1.f / 64.f ? near : far;
}

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
paged_attention_kernel(PagedAttnArgs a, unsigned page_mul, int page_shift, bool out_vec, int t0, int n, float* __restrict__ part,
                       int* __restrict__ counters, int* __restrict__ status) {
  using C = Cfg<DP, NH>;
  constexpr int S = C::STAGES, CH = DP / 8, KS = DP / 16, NT = DP / 16, HEADS = C::HEADS;
  constexpr int VB = NH == 1 && NT % 4 == 0 ? 4 : 2;  // steps of D of the second product side by side, between a weight's two halves
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ long long sm_scan[PA_WARPS];
  __shared__ int sm_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedCache& c = a.cache;
  const int G = a.H / c.Hkv, RT = (G + HEADS - 1) / HEADS, HR = c.Hkv * RT;
  Tokens tk;
  tk.first = reinterpret_cast<long long*>(smem + C::OFF_TOK);
  tk.lo = reinterpret_cast<int*>(tk.first + PAGED_ATTN_CHUNK + 1);
  tk.len = tk.lo + PAGED_ATTN_CHUNK;
  tk.seq = tk.len + PAGED_ATTN_CHUNK;
  // zeros in the query rows that no head fills and, for head sizes between the compiled ones, in the columns that no copy fills
  for (int i = (c.D != DP ? 0 : C::OFF_Q / 16) + tid; i < C::OFF_ACC / 16; i += blockDim.x) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
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
  const int P = (int)min((long long)gridDim.x, max(1ll, U / PA_MIN_SHARE));
  for (int t = blockIdx.x; t < n; t += gridDim.x)
    if (tk.len[t] == 0)
      for (int i = tid; i < a.H * c.D; i += blockDim.x) put((T*)a.out + (t0 + t) * a.o_st + (i / c.D) * a.o_sh + i % c.D, 0.f);
  if (U == 0 || blockIdx.x >= P) return;
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

  // ---- loads: lanes r and r + 16 look up the page of the tile's key r one tile ahead
  const uint32_t sbase = smem_u32(smem);
  const uint32_t my_stage = sbase + warp * C::STAGE;
  const int chunks = c.D >> 3;
  const int r16 = lane & 15;
  long long left = ue - ub;                // units to load
  int ld_items = 0;
  bool ld_new = true;
  unsigned j0, jn;                         // this lane's key of the next tile, the sequence's end
  const int* pages;
  long long head_off;
  auto enter_item = [&]() {
    jn = (unsigned)tk.len[ld.t];
    j0 = (unsigned)tk.lo[ld.t] + (unsigned)ld.v * PA_UNIT + warp * PA_TILE + r16;
    pages = c.table + tk.seq[ld.t] * c.table_stride;
    head_off = (long long)(ld.hr / RT) * c.s_head;
  };
  int pg = -1, row = 0;
  auto look_up = [&]() {
    if (j0 < jn) {
      const unsigned k = __umulhi(2 * j0, page_mul) >> page_shift;  // j0 / page
      row = (int)(j0 - k * c.page);
      pg = __ldcg(pages + k);
    }
  };
  unsigned long long masks = 0;  // 16 bits a stage: which of the tile's keys are there
  auto issue = [&](int stage) {
    if (left > 0) {
      if (pg >= c.n_pages || (pg < 0 && j0 < jn)) {
        pg = -1;
        atomicCAS(status, 0, RT_ERR_BOUNDS);
      }
      const unsigned valid = __ballot_sync(0xffffffffu, pg >= 0) & 0xffffu;
      masks = (masks & ~(0xffffull << (16 * stage))) | (unsigned long long)valid << (16 * stage);
      const uint32_t dst = my_stage + stage * (PA_WARPS * C::STAGE);
      const long long off = pg * c.s_page + row * c.s_row + head_off;
      if (ld_new) {  // this warp's quarter of the item's query rows
        constexpr int QR = HEADS / PA_WARPS;
        const int hk = ld.hr / RT, q0 = (ld.hr - hk * RT) * HEADS + warp * QR;
        const T* const src = (const T*)a.q + (t0 + ld.t) * a.q_st + (long long)(hk * G + q0) * a.q_sh;
        const uint32_t q_dst = sbase + C::OFF_Q + (ld_items % (S + 1)) * C::QBUF + warp * QR * C::ROW;
#pragma unroll
        for (int i = lane; i < QR * CH; i += 32) {
          const int r = i / CH, ch = i % CH;
          if (q0 + r < G && ch < chunks) cp_async16(q_dst + r * C::ROW + ch * 16, src + r * a.q_sh + ch * 8);
        }
        ++ld_items;
      }
      if (valid) {
#pragma unroll
        for (int i = 0; i < PA_TILE * CH / 32; ++i) {
          const int r = (i * 32 + lane) / CH, ch = (i * 32 + lane) % CH;
          const long long o = __shfl_sync(0xffffffffu, off, r) + ch * 8;
          if ((valid >> r & 1) && ch < chunks) {
            cp_async16(dst + r * C::ROW + ch * 16, (const T*)c.k + o);
            cp_async16(dst + (PA_TILE + r) * C::ROW + ch * 16, (const T*)c.v + o);
          }
        }
      }
      --left;
      ld_new = ld.v + 1 == ld.nu;
      j0 += PA_UNIT;
      step(ld);
      pg = -1;
      if (left > 0) {
        if (ld_new) enter_item();
        look_up();
      }
    }
    cp_commit();
  };
  auto arrived = []() {  // this warp's copies of the oldest stage
    cp_wait<S - 1>();
    __syncwarp();
  };
  __syncthreads();  // the zeros are in place
  enter_item();
  look_up();
#pragma unroll
  for (int i = 0; i < S; ++i) issue(i);

  // ---- items
  const float scale2 = a.softcap > 0.f ? a.scale : a.scale * PA_LOG2E;
  const float cap2 = a.softcap * PA_LOG2E, inv_cap = 1.f / a.softcap;  // scale / softcap itself may lie below the 32-bit numbers
  float* acc_buf = reinterpret_cast<float*>(smem + C::OFF_ACC);
  float* sm_m = reinterpret_cast<float*>(smem + C::OFF_ML);
  float* sm_l = sm_m + PA_WARPS * HEADS;
  float* sm_top = sm_l + PA_WARPS * HEADS;  // of the item: maxima, sums, and the sum's inverse (0 of an empty row)
  float* sm_sum = sm_top + HEADS;
  float* sm_inv = sm_sum + HEADS;
  static_assert(2 * HEADS * C::ACC_LD >= PA_WARPS * 32 * 4, "the join's sums fit the merge buffer");
  float* sm_fac = reinterpret_cast<float*>(smem + C::OFF_FAC);  // [32][HEADS] factors of the parts that are joined
  float4* join_buf = reinterpret_cast<float4*>(smem + C::OFF_ACC);
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
    arrived();
    __syncthreads();  // all four warps' query rows have arrived; the merge buffer is free again
    const uint32_t q_lane = sbase + C::OFF_Q + (item % (S + 1)) * C::QBUF + (lane & 7) * C::ROW + (lane >> 3) * 16;
    if constexpr (C::Q_IN_REGS) {
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int k2 = 0; k2 < KS / 2; ++k2) ldsm4(q_lane + h * 8 * C::ROW + k2 * 64, qf[h][k2]);
    }
    for (bool first = true; u < end; ++u, first = false) {
      if (!first) arrived();
      const unsigned mask = (unsigned)(masks >> (16 * stage)) & 0xffffu;
      if (mask) {
        const uint32_t st = stage * (PA_WARPS * C::STAGE);
        const bool all = mask == 0xffffu;
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
            if (a.softcap > 0.f) x = cap2 * tanh_of(x * inv_cap);
            if (!all && !(mask >> ((lane >> 2) + (e < 2 ? 0 : 8)) & 1)) x = -CUDART_INF_F;
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
        uint32_t p[NH][2], rest[NH][2];  // the weights' two parts
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][0][e] = ex2_approx(s[h][0][e] - (m[h][e & 1] == -CUDART_INF_F ? 0.f : m[h][e & 1]));
          l[h][0] += s[h][0][0] + s[h][0][2];
          l[h][1] += s[h][0][1] + s[h][0][3];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t w, r;
            split2<T>(s[h][0][2 * e], s[h][0][2 * e + 1], w, r);
            p[h][e] = transpose8x8(w);
            rest[h][e] = transpose8x8(r);
          }
        }
        const int kk = 2 * (lane & 3);
        const uint32_t keep0 = (mask >> kk & 1 ? 0xffffu : 0u) | (mask >> kk & 2 ? 0xffff0000u : 0u);
        const uint32_t keep1 = (mask >> (kk + 8) & 1 ? 0xffffu : 0u) | (mask >> (kk + 8) & 2 ? 0xffff0000u : 0u);
#pragma unroll
        for (int i0 = 0; i0 < NT; i0 += VB) {
          uint32_t va[VB][4];
#pragma unroll
          for (int i = 0; i < VB; ++i) {
            ldsm4_t(v_lane + st + (i0 + i) * 32, va[i]);
            if (!all) {
              va[i][0] &= keep0;
              va[i][1] &= keep0;
              va[i][2] &= keep1;
              va[i][3] &= keep1;
            }
          }
#pragma unroll
          for (int i = 0; i < VB; ++i)
#pragma unroll
            for (int h = 0; h < NH; ++h) mma16816<T>(o[h][i0 + i], va[i], p[h][0], p[h][1]);
#pragma unroll
          for (int i = 0; i < VB; ++i)
#pragma unroll
            for (int h = 0; h < NH; ++h) mma16816<T>(o[h][i0 + i], va[i], rest[h][0], rest[h][1]);
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
    } else if (warp == 2 && lane < HEADS) {
      const float big = top(lane);
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) x += sm_l[w * HEADS + lane] * factor(sm_m[w * HEADS + lane], big);
      sm_top[lane] = big;
      sm_sum[lane] = x;
      sm_inv[lane] = x == 0.f ? 0.f : 1.f / x;
    }
    __syncthreads();
    T* const out = (T*)a.out + (t0 + t) * a.o_st + (long long)(hk * G + r0) * a.o_sh;
    auto store = [&](int r, int d, float4 x, float f) {
      T* const y = out + r * a.o_sh + d;
      if (out_vec) {
        *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(x.x * f, x.y * f), pack2<T>(x.z * f, x.w * f));
      } else {
        put(y, x.x * f);
        put(y + 1, x.y * f);
        put(y + 2, x.z * f);
        put(y + 3, x.w * f);
      }
    };
    constexpr int D4 = DP / 4;
    const int quads = rows * D4;
    const bool whole = g0 >= ub && g1 <= ue;
    float* const slot = part + ((long long)blockIdx.x * 2 + (g0 >= ub ? 1 : 0)) * C::PART;
    for (int i = tid; i < quads; i += PA_WARPS * 32) {
      const int r = i / D4, d = i % D4 * 4;
      if (d >= c.D) continue;
      const float4 x = *reinterpret_cast<const float4*>(acc_buf + r * C::ACC_LD + d), y = *reinterpret_cast<const float4*>(acc_buf + (HEADS + r) * C::ACC_LD + d);
      const float4 z = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
      if (whole) store(r, d, z, sm_inv[r]);
      else __stcg(reinterpret_cast<float4*>(slot + r * DP + d), z);
    }
    if (!whole) {
      if (tid < rows) {
        __stcg(slot + HEADS * DP + tid, sm_top[tid]);
        __stcg(slot + HEADS * (DP + 1) + tid, sm_sum[tid]);
      }
      const int c0 = (int)(((g0 + 1) * P - 1) / U), c1 = (int)((g1 * P - 1) / U);
      __threadfence();
      __syncthreads();
      if (tid == 0) sm_last = atomicAdd(&counters[c0], 1) == c1 - c0;
      __syncthreads();
      if (sm_last) {
        // Parts in share order: first the item's maxima and sums, a warp a row with the parts over its lanes; then the weighted
        // sum, four values a thread, the parts over the threads that are left and eight loads of each in flight.
        __threadfence();
        const int parts = c1 - c0 + 1;
        auto from = [&](int k) { return part + ((long long)(c0 + k) * 2 + (k == 0 ? 1 : 0)) * C::PART; };
        constexpr int RW = HEADS / PA_WARPS;  // rows of a warp: warp + 4 i
        float big[RW], sum[RW], m0[RW], l0[RW];
#pragma unroll
        for (int i = 0; i < RW; ++i) {  // the lane's first part, all rows at once
          const int r = warp + PA_WARPS * i;
          const bool in = lane < parts && r < rows;
          m0[i] = in ? __ldcg(from(lane) + HEADS * DP + r) : -CUDART_INF_F;
          l0[i] = in ? __ldcg(from(lane) + HEADS * (DP + 1) + r) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < RW; ++i) {
          const int r = warp + PA_WARPS * i;
          big[i] = m0[i];
          if (r < rows)
            for (int k = lane + 32; k < parts; k += 32) big[i] = fmaxf(big[i], __ldcg(from(k) + HEADS * DP + r));
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) big[i] = fmaxf(big[i], __shfl_xor_sync(0xffffffffu, big[i], d));
          sum[i] = l0[i] * factor(m0[i], big[i]);
          if (r < rows)
            for (int k = lane + 32; k < parts; k += 32)
              sum[i] = fmaf(__ldcg(from(k) + HEADS * (DP + 1) + r), factor(__ldcg(from(k) + HEADS * DP + r), big[i]), sum[i]);
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
          if (lane == 0 && r < rows) sm_inv[r] = sum[i] == 0.f ? 0.f : 1.f / sum[i];
        }
        int split = 1;  // threads that share four values
        while (quads * split * 2 <= PA_WARPS * 32 && split * 2 <= parts) split *= 2;
        constexpr int QT = (HEADS * D4 + PA_WARPS * 32 - 1) / (PA_WARPS * 32);  // fours of a thread, where there is one for each
        float4 z[QT];
#pragma unroll
        for (int q = 0; q < QT; ++q) z[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int group = split > 1 ? tid / quads : 0;
        for (int k0 = 0; k0 < parts; k0 += 32) {
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            const int r = warp + PA_WARPS * i, k = k0 + lane;
            const float m = k0 == 0 ? m0[i] : k < parts && r < rows ? __ldcg(from(k) + HEADS * DP + r) : -CUDART_INF_F;
            sm_fac[lane * HEADS + r] = factor(m, big[i]);
          }
          __syncthreads();
          const int end_k = min(parts, k0 + 32);
#pragma unroll
          for (int q = 0; q < QT; ++q) {
            const int i = split > 1 ? tid % quads : tid + q * PA_WARPS * 32;
            const int r = i / D4, d = i % D4 * 4;
            if (i < quads && group < split && d < c.D && (q == 0 || split == 1)) {
#pragma unroll 8
              for (int k = k0 + group; k < end_k; k += split) {
                const float f = sm_fac[(k - k0) * HEADS + r];
                const float4 x = __ldcg(reinterpret_cast<const float4*>(from(k) + r * DP + d));
                z[q] = make_float4(fmaf(x.x, f, z[q].x), fmaf(x.y, f, z[q].y), fmaf(x.z, f, z[q].z), fmaf(x.w, f, z[q].w));
              }
            }
          }
          __syncthreads();
        }
        if (split == 1) {
#pragma unroll
          for (int q = 0; q < QT; ++q) {
            const int i = tid + q * PA_WARPS * 32, d = i % D4 * 4;
            if (i < quads && d < c.D) store(i / D4, d, z[q], sm_inv[i / D4]);
          }
        } else {
          if (group < split) join_buf[tid] = z[0];
          __syncthreads();
          if (tid < quads && tid % D4 * 4 < c.D) {
            float4 x = join_buf[tid];
            for (int g = 1; g < split; ++g) {
              const float4 y = join_buf[g * quads + tid];
              x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
            }
            store(tid / D4, tid % D4 * 4, x, sm_inv[tid / D4]);
          }
        }
        if (tid == 0) counters[c0] = 0;  // for the next launch that uses this workspace
      }
    }
  }
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
  const bool out_vec = a.o_st % 4 == 0 && a.o_sh % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 8 == 0;
  dispatch(a, [&](auto type, auto dp, auto nh) {
    constexpr int DP = decltype(dp)::value, NH = decltype(nh)::value;
    for (int t0 = 0; t0 < a.n_tok; t0 += PAGED_ATTN_CHUNK) {
      launch_pdl(paged_attention_kernel<decltype(type), DP, NH>, dim3(p.grid), dim3(PA_WARPS * 32), Cfg<DP, NH>::SMEM, s, a, mul, shift, out_vec, t0,
                 std::min(a.n_tok - t0, PAGED_ATTN_CHUNK), part, counters, status);
      RT_LAUNCH_CHECK();
    }
    return 0;
  });
}

}  // namespace rt
