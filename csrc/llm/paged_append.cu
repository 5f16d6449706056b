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

#include <type_traits>

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
  const double halves = (double)pos * (double)inv_freq * 0.31830988618379067154;  // 1 / pi
  sincospif((float)(halves - 2.0 * rint(0.5 * halves)), sn, cs);
}

// Where a token's keys and values go (element offset of head 0 in the cache), -1 for padded and refused tokens.
__device__ __forceinline__ long long slot_of(const PagedCache& c, int p, int s, bool report, int* status) {
  if (s == -1) return -1;
  const int k = p / c.page;
  if (p >= 0 && s >= 0 && s < c.n_seq && k < c.max_pages) {
    const int page = __ldcg(c.table + s * c.table_stride + k);
    if (page >= 0 && page < c.n_pages) return page * c.s_page + (p - k * c.page) * c.s_row;
  }
  if (report) atomicCAS(status, 0, RT_ERR_BOUNDS);
  return -1;
}

// Two 32-bit values in a register pair, and the packed multiply-add that takes such pairs.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 swap(F2 a) {
  float lo, hi;
  unpair(a, lo, hi);
  return f2(hi, lo);
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
template <typename T> __device__ __forceinline__ F2 widen(uint32_t r);
template <> __device__ __forceinline__ F2 widen<__half>(uint32_t r) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&r));
  return f2(v.x, v.y);
}
template <> __device__ __forceinline__ F2 widen<__nv_bfloat16>(uint32_t r) { return f2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u)); }
template <typename T> __device__ __forceinline__ uint32_t narrow(F2 a) {
  float lo, hi;
  unpair(a, lo, hi);
  return pack_2x16<std::is_same<T, __half>::value>(lo, hi);
}

constexpr int AP_WARPS = 4;
constexpr int AP_BATCH = 2;      // rows a lane has in flight

template <int N> struct Raw;     // N 16-bit values as they lie in memory
template <> struct Raw<4> { using V = uint2; };
template <> struct Raw<8> { using V = uint4; };

// A warp takes one token and a share of its head rows.  LPR lanes hold a row, 2 SIDE values each: SIDE rotation pairs, both
// sides, so a row is read and written in pieces of SIDE values and nothing moves between lanes but the norm's sum; the lane's
// pairs are the same for every head, so its coefficients (cosine and sine times the norm's weights) stay in registers:
//   a <- r (a wa cos - b wb sin),  b <- r (a wa sin + b wb cos),  r = rsqrt(mean + eps) or 1
// in packed 32-bit pairs.  Cosines and sines are computed once a warp, one pair a lane at a time, while the first rows load.
// Bound by bytes where there are many tokens, with waits for loads beside (2.8 waves of CTAs): 8192 tokens of 32 + 2 x 8 heads of 128,
// normalised, move 201 MB in 40 us (5.0 TB/s, 0.76 of a plain copy's rate).
// Four values a side 43 us, coefficients in shared memory 51 us, a warp a row (the general kernel) 180 us.
template <typename T, bool INTERLEAVED, int LPR, int SIDE>
__global__ void __launch_bounds__(AP_WARPS * 32, SIDE == 4 ? 8 : 5) paged_append_vec_kernel(PagedAppendArgs a, int parts, int* status) {
  using V = typename Raw<SIDE>::V;
  constexpr int RPW = 32 / LPR, N2 = SIDE / 2;                     // rows of a step, packed pairs of a side
  __shared__ float2 sm_turn[AP_WARPS][LPR * SIDE];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * AP_WARPS + warp;
  const int t = (int)(w / parts), part = (int)(w % parts);
  if (t >= a.n_tok) return;
  const int D = a.cache.D, half = a.rot >> 1, H = a.H, Hkv = a.cache.Hkv;
  const int p = __ldcg(a.pos + t), s = a.seq ? __ldcg(a.seq + t) : t;
  const int i = lane % LPR, hl = lane / LPR;
  const bool in_row = i * 2 * SIDE < D;
  // places of this lane's values: the two sides of its pairs (one run where pairs are adjacent or do not turn)
  const bool turns = i * SIDE < half;
  const int d0 = INTERLEAVED || !turns ? i * 2 * SIDE : i * SIDE, gap = INTERLEAVED || !turns ? SIDE : half;
  auto load = [&](const T* src, long long s_inc, int h, int h_step, int heads, V (&r)[AP_BATCH][2]) {
#pragma unroll
    for (int b = 0; b < AP_BATCH; ++b) {
      r[b][0] = r[b][1] = V();
      if (in_row && h + b * h_step < heads) {
        r[b][0] = *reinterpret_cast<const V*>(src + b * s_inc);
        r[b][1] = *reinterpret_cast<const V*>(src + b * s_inc + gap);
      }
    }
  };
  // rows h of one kind, RPW a step, every parts-th step from (part - shift) mod parts on
  const int h_step = parts * RPW;
  auto first_row = [&](int shift) {
    int step = (part - shift) % parts;
    if (step < 0) step += parts;
    return step * RPW;
  };
  const T* const q_src = (const T*)a.q + t * a.q_st + d0 + (long long)(first_row(0) + hl) * a.q_sh;
  V raw[AP_BATCH][2];
  load(q_src, h_step * a.q_sh, first_row(0) + hl, h_step, H, raw);

  const long long slot = slot_of(a.cache, p, s, part == 0 && lane == 0, status);
  if (slot >= 0) {
    for (int k = lane; k < half; k += 32) {
      float cs, sn;
      rotation(p, a.inv_freq[k], &cs, &sn);
      sm_turn[warp][k] = make_float2(cs, sn);
    }
  }
  __syncwarp();
  const float inv_d = 1.f / D;

  auto rows_of = [&](auto rotated, int heads, int h0, const T* src, long long s_sh, T* out, long long o_sh, T* dst, long long d_sh, const T* wt) {
    constexpr bool ROT = decltype(rotated)::value;
    if (h0 >= heads) return;
    F2 k0[SIDE], k1[SIDE];
    if constexpr (ROT) {
      float wv[2 * SIDE], cs[SIDE], sn[SIDE];
#pragma unroll
      for (int e = 0; e < SIDE; ++e) {
        const float2 x = slot >= 0 && i * SIDE + e < half ? sm_turn[warp][i * SIDE + e] : make_float2(1.f, 0.f);
        cs[e] = x.x;
        sn[e] = x.y;
        wv[e] = wt && in_row ? to_f(wt[d0 + e]) : 1.f;
        wv[SIDE + e] = wt && in_row ? to_f(wt[d0 + gap + e]) : 1.f;
      }
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < SIDE; ++e) {  // (a, b) <- (a, b) k0 + (b, a) k1
          k0[e] = f2(wv[2 * e] * cs[e], wv[2 * e + 1] * cs[e]);
          k1[e] = f2(-wv[2 * e + 1] * sn[e], wv[2 * e] * sn[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < N2; ++e) {  // a <- a k0[e] + b k1[e],  b <- a k1[N2 + e] + b k0[N2 + e]
          const int x = 2 * e, y = x + 1;
          k0[e] = f2(wv[x] * cs[x], wv[y] * cs[y]);
          k1[e] = f2(-wv[SIDE + x] * sn[x], -wv[SIDE + y] * sn[y]);
          k1[N2 + e] = f2(wv[x] * sn[x], wv[y] * sn[y]);
          k0[N2 + e] = f2(wv[SIDE + x] * cs[x], wv[SIDE + y] * cs[y]);
        }
      }
    }
    const long long s_inc = h_step * s_sh, o_inc = h_step * o_sh, d_inc = h_step * d_sh;
    if (out) out += (h0 + hl) * o_sh + d0;
    dst = slot >= 0 && dst ? dst + (h0 + hl) * d_sh + d0 : nullptr;
    while (true) {
#pragma unroll
      for (int b = 0; b < AP_BATCH; ++b) {
        V(&r)[2] = raw[b];
        if constexpr (ROT) {
          F2 x[SIDE], y[SIDE];
          const uint32_t* const words = reinterpret_cast<const uint32_t*>(&r[0]);
#pragma unroll
          for (int e = 0; e < SIDE; ++e) x[e] = widen<T>(words[e]);
          if constexpr (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < SIDE; ++e) y[e] = fma2(x[e], k0[e], mul2(swap(x[e]), k1[e]));
          } else {
#pragma unroll
            for (int e = 0; e < N2; ++e) {
              y[e] = fma2(x[e], k0[e], mul2(x[N2 + e], k1[e]));
              y[N2 + e] = fma2(x[N2 + e], k0[N2 + e], mul2(x[e], k1[N2 + e]));
            }
          }
          if (wt) {
            F2 ss = mul2(x[0], x[0]);
#pragma unroll
            for (int e = 1; e < SIDE; ++e) ss = fma2(x[e], x[e], ss);
            float lo, hi;
            unpair(ss, lo, hi);
            lo += hi;
#pragma unroll
            for (int o = LPR >> 1; o > 0; o >>= 1) lo += __shfl_xor_sync(0xffffffffu, lo, o);
            const float n = rsqrtf(fmaf(lo, inv_d, a.eps));
#pragma unroll
            for (int e = 0; e < SIDE; ++e) y[e] = mul2(y[e], f2(n, n));
          }
          uint32_t* const put = reinterpret_cast<uint32_t*>(&r[0]);
#pragma unroll
          for (int e = 0; e < SIDE; ++e) put[e] = slot >= 0 ? narrow<T>(y[e]) : 0u;  // a padded or refused token: zeros, nothing appended
        }
        if (in_row && h0 + hl + b * h_step < heads) {
          if (out) {
            *reinterpret_cast<V*>(out) = r[0];
            *reinterpret_cast<V*>(out + gap) = r[1];
          }
          if (dst) {
            *reinterpret_cast<V*>(dst) = r[0];
            *reinterpret_cast<V*>(dst + gap) = r[1];
          }
        }
        if (out) out += o_inc;
        if (dst) dst += d_inc;
      }
      h0 += AP_BATCH * h_step;
      if (h0 >= heads) return;
      src += AP_BATCH * s_inc;
      load(src, s_inc, h0 + hl, h_step, heads, raw);
    }
  };
  rows_of(std::true_type(), H, first_row(0), q_src, a.q_sh, (T*)a.q_out + t * a.qo_st, a.qo_sh, (T*)nullptr, 0, (const T*)a.q_norm);
  const int q_steps = (H + RPW - 1) / RPW, k_steps = (Hkv + RPW - 1) / RPW;
  const int hk = first_row(q_steps), hv = first_row(q_steps + k_steps);
  const T* const k_src = (const T*)a.k + t * a.k_st + d0 + (long long)(hk + hl) * a.k_sh;
  load(k_src, h_step * a.k_sh, hk + hl, h_step, Hkv, raw);
  rows_of(std::true_type(), Hkv, hk, k_src, a.k_sh, a.k_out ? (T*)a.k_out + t * a.ko_st : nullptr, a.ko_sh, (T*)a.cache.k + slot, a.cache.s_head,
          (const T*)a.k_norm);
  const T* const v_src = (const T*)a.v + t * a.v_st + d0 + (long long)(hv + hl) * a.v_sh;
  load(v_src, h_step * a.v_sh, hv + hl, h_step, Hkv, raw);
  rows_of(std::false_type(), Hkv, hv, v_src, a.v_sh, (T*)nullptr, 0, (T*)a.cache.v + slot, a.cache.s_head, (const T*)nullptr);
}

template <typename T, bool INTERLEAVED, int LPR, int SIDE>
void launch_vec(const PagedAppendArgs& a, int* status, cudaStream_t s) {
  constexpr int RPW = 32 / LPR;
  // A token's rows go to several warps while there are fewer than eight warps an SM; each repeats the token's cosines and
  // look-ups, which costs more than it gains from there on (8192 tokens: 40 us with one warp a token, 48 with two, 57 with three).
  const long long steps = (a.H + RPW - 1) / RPW + 2 * ((a.cache.Hkv + RPW - 1) / RPW);
  const long long want = (8ll * sm_count(current_device()) + a.n_tok - 1) / a.n_tok;
  const int parts = (int)(want < steps ? want : steps);
  launch_pdl(paged_append_vec_kernel<T, INTERLEAVED, LPR, SIDE>, dim3((unsigned)(((long long)a.n_tok * parts + AP_WARPS - 1) / AP_WARPS)),
             dim3(AP_WARPS * 32), 0, s, a, parts, status);
}
template <typename T, bool INTERLEAVED, int SIDE>
void launch_vec_width(const PagedAppendArgs& a, int* status, cudaStream_t s) {
  const int lanes = (a.cache.D + 2 * SIDE - 1) / (2 * SIDE);
  if (lanes <= 4) launch_vec<T, INTERLEAVED, 4, SIDE>(a, status, s);
  else if (lanes <= 8) launch_vec<T, INTERLEAVED, 8, SIDE>(a, status, s);
  else if (lanes <= 16) launch_vec<T, INTERLEAVED, 16, SIDE>(a, status, s);
  else launch_vec<T, INTERLEAVED, 32, SIDE>(a, status, s);
}
template <typename T, int SIDE>
void launch_vec_order(const PagedAppendArgs& a, int* status, cudaStream_t s) {
  if (a.interleaved) launch_vec_width<T, true, SIDE>(a, status, s);
  else launch_vec_width<T, false, SIDE>(a, status, s);
}

// Any head size, stride and alignment: one warp per (token, head row), q heads, then k heads, then v heads.
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
  const int p = __ldcg(a.pos + t), s = a.seq ? __ldcg(a.seq + t) : t;
  const long long slot = slot_of(a.cache, p, s, h == 0 && lane == 0, status);
  const T* src = kind == 0 ? (const T*)a.q + t * a.q_st + hh * a.q_sh
                           : kind == 1 ? (const T*)a.k + t * a.k_st + hh * a.k_sh : (const T*)a.v + t * a.v_st + hh * a.v_sh;
  T* out = kind == 0 ? (T*)a.q_out + t * a.qo_st + hh * a.qo_sh
                     : kind == 1 && a.k_out ? (T*)a.k_out + t * a.ko_st + hh * a.ko_sh : nullptr;
  T* dst = kind == 0 || slot < 0 ? nullptr : (T*)(kind == 1 ? a.cache.k : a.cache.v) + slot + hh * a.cache.s_head;
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
  int* status = status_word(current_device());
  const long long rows = (long long)a.H + 2 * a.cache.Hkv;
  const PagedCache& c = a.cache;
  // Pieces of `side` values: whole ones on either side of the rotation pairs, rows that start on their boundaries, at most 32 lanes a row.
  auto fits = [&](int side) {
    auto even = [&](const void* p, long long st, long long sh) { return reinterpret_cast<uintptr_t>(p) % (2 * side) == 0 && st % side == 0 && sh % side == 0; };
    return c.D % (2 * side) == 0 && c.D <= 64 * side && a.rot % (2 * side) == 0 && even(a.q, a.q_st, a.q_sh) && even(a.k, a.k_st, a.k_sh) &&
           even(a.v, a.v_st, a.v_sh) && even(a.q_out, a.qo_st, a.qo_sh) && even(a.k_out, a.ko_st, a.ko_sh) && even(c.k, c.s_page, c.s_head) &&
           even(c.v, c.s_row, 0);
  };
  // Tokens of few values are bound by the look-ups before their rows, so pieces of four, whose registers let 32 warps an SM run instead
  // of 20, serve them better (107264 tokens of 8 + 2 heads of 32: 123 us, 162 with eight; 76775 of 4 + 2 of 96 112, 149); tokens of
  // 32 + 16 heads of 128 40.2 with four, 38.0 with eight; 12 + 24 of 64 alike.
  const bool light = rows * c.D < 2048 && fits(4);
  if (!light && fits(8)) {
    if (a.dtype == DT_F16) launch_vec_order<__half, 8>(a, status, s);
    else launch_vec_order<__nv_bfloat16, 8>(a, status, s);
  } else if (fits(4)) {
    if (a.dtype == DT_F16) launch_vec_order<__half, 4>(a, status, s);
    else launch_vec_order<__nv_bfloat16, 4>(a, status, s);
  } else {
    const dim3 grid((unsigned)((a.n_tok * rows + 7) / 8)), block(256);
    if (a.dtype == DT_F16) launch_pdl(paged_append_kernel<__half>, grid, block, 0, s, a, status);
    else launch_pdl(paged_append_kernel<__nv_bfloat16>, grid, block, 0, s, a, status);
  }
  RT_LAUNCH_CHECK();
}

}  // namespace rt
