// Per-head RMSNorm of queries and keys with the position rotation in the same pass, for MI355X
// (gfx950): what stands between qkv_proj and attention.
//
//   h = x * rsqrt(mean(x^2) + eps) * w           over the D values of a head (w: 1 when absent)
//   (h_a, h_b) -> (h_a c - h_b s, h_b c + h_a s)   for the R/2 pairs of the first R values
//
// with (c, s) the row of the token's position in the cos|sin table; the pairs are (i, i + R/2), or
// (2i, 2i + 1) interleaved, and values from R on are normalized only.  All of it in fp32 with one
// rounding at the end.
//
// What bounds it: HBM (every value is read and written once, 4 bytes of bf16).  A lane owns two runs of V
// values R/2 apart, so both members of every pair of either kind are its own and nothing but the sum
// of squares crosses lanes (L lanes a head, a power of two: DPP steps), each load is 16 bytes, and a
// head that is written over its own input is read whole by the lanes that write it.  A wave takes
// 64/L heads at a time of one token, whose cos, sin and the two weights stay in its registers; they
// are loaded 16 bytes at a time, with no choice of type inside (a value at a time, a token of 16 + 8
// heads takes 6.2 us; so 3.3).  4096 tokens of 32 + 8 heads of 128: 16.2 us over the same rows again and
// again (5.2 TB/s), 23.2 where rows and outputs change from launch to launch.
#include <algorithm>

#include "i8l_common.h"

namespace i8l {

namespace {

struct QkArgs {
  const void *q, *k;
  void *qo, *ko;
  int64_t q_ts, q_hs, k_ts, k_hs, qo_ts, qo_hs, ko_ts, ko_hs;   // token and head strides, elements
  const void *qw, *kw;                                          // NULL: no weight
  const void *cs, *pos;
  int64_t max_pos, T;
  int hq, hk, D, R, w_dtype, cs_dtype, pos64, parts;            // parts: waves a token
  float eps;
};

__device__ __forceinline__ float load_f(const void* p, int dt, int64_t i) {
  if (dt == I8L_F32) return ((const float*)p)[i];
  return act_to_f32(((const uint16_t*)p)[i], dt);
}

// The token's row of the table; a position outside it has none (its pairs become NaN).
__device__ __forceinline__ int64_t table_row(const QkArgs& a, int64_t t) {
  const int64_t p = a.pos64 ? ((const int64_t*)a.pos)[t] : ((const int32_t*)a.pos)[t];
  return p >= 0 && p < a.max_pos ? p : -1;
}

// Sum over each aligned group of L lanes (a power of two, uniform).
__device__ __forceinline__ float lanes_sum(float v, int L) {
  v += __int_as_float(dpp_i<kQuadSwap1>(__float_as_int(v)));
  v += __int_as_float(dpp_i<kQuadSwap2>(__float_as_int(v)));
  if (L >= 8) v += __int_as_float(dpp_i<kHalfMirror>(__float_as_int(v)));
  if (L >= 16) v += __int_as_float(dpp_i<kRowMirror>(__float_as_int(v)));
  if (L >= 32)
    v += __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), kSwizzleXor16));
  if (L >= 64) v += __shfl_xor(v, 32);
  return v;
}

// V consecutive 16-bit values (V = 8 or 4), as loaded.
template <int V>
struct Run {
  uint32_t w[V / 2];
};
template <int V>
__device__ __forceinline__ Run<V> load_run(const uint16_t* p) {
  Run<V> r;
  if constexpr (V == 8) {
    const uint4 v = *(const uint4*)p;
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else {
    const uint2 v = *(const uint2*)p;
    r.w[0] = v.x, r.w[1] = v.y;
  }
  return r;
}
template <int V, int DT>
__device__ __forceinline__ void store_run(uint16_t* p, const float (&v)[V]) {
  uint32_t w[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) w[i] = f32x2_to_act2<DT>(v[2 * i], v[2 * i + 1]);
  if constexpr (V == 8) *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
  else *(uint2*)p = make_uint2(w[0], w[1]);
}

// N consecutive values of a table or weight as floats, by one load of 16 bytes or two; F32: of fp32,
// else of the 16-bit dtype dt.
template <int N, bool F32>
__device__ __forceinline__ void load_floats(const void* p, int dt, int64_t at, float (&o)[N]) {
  if constexpr (F32) {
    const float* f = (const float*)p + at;
    if constexpr (N == 2) {
      const float2 v = *(const float2*)f;
      o[0] = v.x, o[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 v = *(const float4*)(f + i);
        o[i] = v.x, o[i + 1] = v.y, o[i + 2] = v.z, o[i + 3] = v.w;
      }
    }
  } else {
    const uint16_t* h = (const uint16_t*)p + at;
    uint32_t w[N / 2];
    if constexpr (N == 2) {
      w[0] = *(const uint32_t*)h;
    } else {
      const Run<N> r = load_run<N>(h);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = r.w[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = act_to_f32(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu, dt);
  }
}

// L lanes a head: the first R / 2V own the rotated runs [V j, V j + V) and R/2 further, the next
// ones two runs of the rest, the others none.  C32: the table is fp32; W32: the weights are (or there
// is none).
template <int DT, int V, bool INTER, bool C32, bool W32>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QkArgs a, int L, int logL) {
  const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = wave / (uint32_t)a.parts;
  if (t >= a.T) return;
  const int part = wave % (uint32_t)a.parts;
  const int64_t row = table_row(a, t);
  const int lane = threadIdx.x & 63, j = lane & (L - 1), sub = lane >> logL;
  const int per = 64 >> logL, heads = a.hq + a.hk, groups = (heads + per - 1) / per;
  const int rl = a.R / (2 * V);
  const bool turned = j < rl;
  const int d0 = turned ? V * j : a.R + 2 * V * (j - rl);
  const int d1 = turned ? d0 + a.R / 2 : d0 + V;
  const bool in0 = d0 < a.D, in1 = d1 < a.D;

  const uint16_t *q = (const uint16_t*)a.q + t * a.q_ts, *k = (const uint16_t*)a.k + t * a.k_ts;
  uint16_t *qo = (uint16_t*)a.qo + t * a.qo_ts, *ko = (uint16_t*)a.ko + t * a.ko_ts;
  struct Head {
    int i;        // among the queries, or the keys
    bool q, on;
  };
  auto head_at = [&](int g) {
    Head h;
    h.i = g * per + sub;
    h.on = g < groups && h.i < heads;
    h.q = h.i < a.hq;
    if (!h.q) h.i -= a.hq;
    return h;
  };
  auto load = [&](const Head& h, Run<V>(&r)[2]) {
    const uint16_t* p = (h.q ? q : k) + h.i * (int)(h.q ? a.q_hs : a.k_hs);
    r[0] = Run<V>{}, r[1] = Run<V>{};
    if (h.on && in0) r[0] = load_run<V>(p + d0);
    if (h.on && in1) r[1] = load_run<V>(p + d1);
  };

  Head h = head_at(part);
  Run<V> raw[2];
  load(h, raw);
  float wq[2][V], wk[2][V];
#pragma unroll
  for (int i = 0; i < V; ++i) wq[0][i] = wq[1][i] = wk[0][i] = wk[1][i] = 1.0f;
  if (a.qw) {
    if (in0) load_floats<V, W32>(a.qw, a.w_dtype, d0, wq[0]);
    if (in1) load_floats<V, W32>(a.qw, a.w_dtype, d1, wq[1]);
  }
  if (a.kw) {
    if (in0) load_floats<V, W32>(a.kw, a.w_dtype, d0, wk[0]);
    if (in1) load_floats<V, W32>(a.kw, a.w_dtype, d1, wk[1]);
  }
  // the token's angles; the two runs have the same ones, or V/2 each when interleaved
  float c[V] = {}, s[V] = {};
  if (turned) {
    const int64_t at = row * a.R;
    if (row < 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = s[i] = __builtin_nanf("");
    } else if constexpr (INTER) {
      float c0[V / 2], c1[V / 2], s0[V / 2], s1[V / 2];
      load_floats<V / 2, C32>(a.cs, a.cs_dtype, at + d0 / 2, c0);
      load_floats<V / 2, C32>(a.cs, a.cs_dtype, at + d1 / 2, c1);
      load_floats<V / 2, C32>(a.cs, a.cs_dtype, at + a.R / 2 + d0 / 2, s0);
      load_floats<V / 2, C32>(a.cs, a.cs_dtype, at + a.R / 2 + d1 / 2, s1);
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        c[i] = c0[i], c[V / 2 + i] = c1[i], s[i] = s0[i], s[V / 2 + i] = s1[i];
    } else {
      load_floats<V, C32>(a.cs, a.cs_dtype, at + d0, c);
      load_floats<V, C32>(a.cs, a.cs_dtype, at + a.R / 2 + d0, s);
    }
  }
  for (int g = part; g < groups; g += a.parts) {
    const Head next = head_at(g + a.parts);
    Run<V> ahead[2];
    load(next, ahead);
    float x[2][V], sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[r][i] = act_to_f32<DT>(i % 2 ? raw[r].w[i / 2] >> 16 : raw[r].w[i / 2] & 0xffffu);
        sum = __builtin_fmaf(x[r][i], x[r][i], sum);
      }
    sum = lanes_sum(sum, L);
    const float rs = 1.0f / __builtin_sqrtf(sum / (float)a.D + a.eps);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) x[r][i] = x[r][i] * rs * (h.q ? wq[r][i] : wk[r][i]);
    if (turned) {   // (an angle of 0 would not do: a NaN or an infinity times its sine is a NaN)
      if constexpr (INTER) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const float ca = c[r * (V / 2) + i / 2], sa = s[r * (V / 2) + i / 2];
            const float u = x[r][i], v = x[r][i + 1];
            x[r][i] = __builtin_fmaf(u, ca, -(v * sa));
            x[r][i + 1] = __builtin_fmaf(v, ca, u * sa);
          }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = x[0][i], v = x[1][i];
          x[0][i] = __builtin_fmaf(u, c[i], -(v * s[i]));
          x[1][i] = __builtin_fmaf(v, c[i], u * s[i]);
        }
      }
    }
    uint16_t* p = (h.q ? qo : ko) + h.i * (int)(h.q ? a.qo_hs : a.ko_hs);
    if (h.on && in0) store_run<V, DT>(p + d0, x[0]);
    if (h.on && in1) store_run<V, DT>(p + d1, x[1]);
    h = next;
    raw[0] = ahead[0], raw[1] = ahead[1];
  }
}

// Any sizes, strides and alignment: a wave a head, a lane a pair (or a value past R) at a time.
template <int DT>
__global__ void __launch_bounds__(256) qk_norm_rope_any_kernel(QkArgs a, int inter) {
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int heads = a.hq + a.hk, lane = threadIdx.x & 63;
  const int64_t t = wave / heads;
  if (t >= a.T) return;
  int i = (int)(wave % heads);
  const bool q = i < a.hq;
  if (!q) i -= a.hq;
  const uint16_t* in = (const uint16_t*)(q ? a.q : a.k) + t * (q ? a.q_ts : a.k_ts) +
                       (int64_t)i * (q ? a.q_hs : a.k_hs);
  uint16_t* out = (uint16_t*)(q ? a.qo : a.ko) + t * (q ? a.qo_ts : a.ko_ts) +
                  (int64_t)i * (q ? a.qo_hs : a.ko_hs);
  const void* w = q ? a.qw : a.kw;
  const int64_t row = table_row(a, t);
  float sum = 0.0f;
  for (int d = lane; d < a.D; d += 64) {
    const float x = act_to_f32<DT>(in[d]);
    sum = __builtin_fmaf(x, x, sum);
  }
  sum = lanes_sum(sum, 64);   // past here every lane has read the head: it may be written over
  const float rs = 1.0f / __builtin_sqrtf(sum / (float)a.D + a.eps);
  auto normed = [&](int d) {
    return act_to_f32<DT>(in[d]) * rs * (w ? load_f(w, a.w_dtype, d) : 1.0f);
  };
  const int half = a.R / 2;
  for (int p = lane; p < half; p += 64) {
    const int d0 = inter ? 2 * p : p, d1 = inter ? d0 + 1 : p + half;
    const float c = row >= 0 ? load_f(a.cs, a.cs_dtype, row * a.R + p) : __builtin_nanf("");
    const float s = row >= 0 ? load_f(a.cs, a.cs_dtype, row * a.R + half + p) : __builtin_nanf("");
    const float u = normed(d0), v = normed(d1);
    out[d0] = f32_to_act<DT>(__builtin_fmaf(u, c, -(v * s)));
    out[d1] = f32_to_act<DT>(__builtin_fmaf(v, c, u * s));
  }
  for (int d = a.R + lane; d < a.D; d += 64) out[d] = f32_to_act<DT>(normed(d));
}

// Waves that fill the card: a token's heads are spread over more waves until there are this many (256
// CUs, 4 SIMDs, 4 waves a SIMD).  More repeat the token's angles and weights: 2048 tokens of 16 + 8
// heads 8.7 us, at four times the waves 10.1; 4096 of 32 + 8 19.7, at twice 20.3, at four times 23.8
// (rows that change from launch to launch).
constexpr int64_t kQkWaves = 4096;

template <int DT, int V, bool INTER>
void launch_qk(QkArgs a, int L, hipStream_t st) {
  int logL = 0;
  while ((1 << logL) < L) ++logL;
  const int per = 64 / L, groups = (a.hq + a.hk + per - 1) / per;
  a.parts = (int)std::min<int64_t>(groups, std::max<int64_t>(1, (kQkWaves + a.T - 1) / a.T));
  const bool w32 = a.w_dtype == I8L_F32 || !(a.qw || a.kw);
  auto kern = a.cs_dtype == I8L_F32 ? (w32 ? qk_norm_rope_kernel<DT, V, INTER, true, true>
                                           : qk_norm_rope_kernel<DT, V, INTER, true, false>)
                                    : (w32 ? qk_norm_rope_kernel<DT, V, INTER, false, true>
                                           : qk_norm_rope_kernel<DT, V, INTER, false, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)((a.T * a.parts + 3) / 4)), dim3(256), 0, st, a, L, logL);
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int i8l_qk_norm_rope(const void* q, int64_t q_ts, int64_t q_hs, const void* k,
                                int64_t k_ts, int64_t k_hs, void* q_out, int64_t qo_ts,
                                int64_t qo_hs, void* k_out, int64_t ko_ts, int64_t ko_hs,
                                const void* q_weight, const void* k_weight, int32_t w_dtype,
                                float eps, const void* cos_sin, int32_t cs_dtype, int64_t max_pos,
                                const void* positions, int32_t pos_bits, int64_t T, int64_t Hq,
                                int64_t Hk, int64_t D, int64_t R, int32_t interleaved,
                                int32_t act_dtype, void* stream) {
  if (T < 0 || Hq < 0 || Hk < 0 || D <= 0 || R < 2 || R > D || R % 2 || max_pos < 0) {
    set_error("qk_norm_rope: bad sizes T=%lld heads %lld + %lld of %lld, %lld rotated", (long long)T,
              (long long)Hq, (long long)Hk, (long long)D, (long long)R);
    return I8L_INVALID_ARG;
  }
  if (act_dtype != I8L_BF16 && act_dtype != I8L_F16) {
    set_error("qk_norm_rope: queries and keys must be bf16 or fp16");
    return I8L_UNSUPPORTED;
  }
  auto float_dt = [](int dt) { return dt == I8L_BF16 || dt == I8L_F16 || dt == I8L_F32; };
  if (!float_dt(cs_dtype) || ((q_weight || k_weight) && !float_dt(w_dtype))) {
    set_error("qk_norm_rope: the weights and the table must be bf16, fp16 or fp32");
    return I8L_UNSUPPORTED;
  }
  if (pos_bits != 32 && pos_bits != 64) {
    set_error("qk_norm_rope: positions of 32 or 64 bits, not %d", pos_bits);
    return I8L_INVALID_ARG;
  }
  if (D > 65536 || Hq + Hk > 65536 || T * (Hq + Hk) > INT32_MAX) {
    set_error("qk_norm_rope: %lld tokens of %lld + %lld heads of %lld: too large", (long long)T,
              (long long)Hq, (long long)Hk, (long long)D);
    return I8L_UNSUPPORTED;
  }
  if (T == 0 || Hq + Hk == 0) return I8L_OK;
  if (!operands_ok("qk_norm_rope", {cos_sin, positions}) ||
      (Hq && !operands_ok("qk_norm_rope", {q, q_out})) ||
      (Hk && !operands_ok("qk_norm_rope", {k, k_out})))
    return I8L_INVALID_ARG;
  QkArgs a{q, k, q_out, k_out, q_ts, q_hs, k_ts, k_hs, qo_ts, qo_hs, ko_ts, ko_hs, q_weight,
           k_weight, cos_sin, positions, max_pos, T, (int)Hq, (int)Hk, (int)D, (int)R, w_dtype,
           cs_dtype, pos_bits == 64, 1, eps};
  // every run of V values aligned: its pointers and strides, and the dimensions it starts at
  auto runs = [&](int V) {
    const int64_t b = 2 * V;
    auto at = [&](const void* p, int64_t ts, int64_t hs, int64_t n) {
      return !n || ((uintptr_t)p % b == 0 && ts % V == 0 && hs % V == 0 && hs >= 0 &&
                    (n - 1) * hs + D < INT32_MAX);
    };
    auto whole = [&](const void* p) { return (uintptr_t)p % 16 == 0; };
    const int64_t lanes = R / (2 * V) + (D - R + 2 * V - 1) / (2 * V);
    return R % (2 * V) == 0 && D % V == 0 && lanes <= 64 && at(q, q_ts, q_hs, Hq) &&
           at(q_out, qo_ts, qo_hs, Hq) && at(k, k_ts, k_hs, Hk) && at(k_out, ko_ts, ko_hs, Hk) &&
           whole(cos_sin) && whole(q_weight) && whole(k_weight);
  };
  const int V = runs(8) ? 8 : runs(4) ? 4 : 0;
  // a grid's threads stay below 2^32, so its waves at 2^26 less a workgroup's: as many as tokens from
  // kQkWaves tokens on (launch_qk), else as heads
  if (T * (V ? 1 : Hq + Hk) > ((int64_t)1 << 26) - 4) {
    set_error("qk_norm_rope: %lld tokens of %lld + %lld heads of %lld: too large", (long long)T,
              (long long)Hq, (long long)Hk, (long long)D);
    return I8L_UNSUPPORTED;
  }
  const hipStream_t st = (hipStream_t)stream;
  if (V) {
    const int lanes = (int)(R / (2 * V) + (D - R + 2 * V - 1) / (2 * V));
    int L = 4;
    while (L < lanes) L *= 2;
    auto go = [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      if (V == 8) interleaved ? launch_qk<DT, 8, true>(a, L, st) : launch_qk<DT, 8, false>(a, L, st);
      else interleaved ? launch_qk<DT, 4, true>(a, L, st) : launch_qk<DT, 4, false>(a, L, st);
    };
    if (act_dtype == I8L_BF16) go(std::integral_constant<int, I8L_BF16>{});
    else go(std::integral_constant<int, I8L_F16>{});
  } else {
    const dim3 grid((unsigned)((T * (Hq + Hk) + 3) / 4));
    if (act_dtype == I8L_BF16)
      hipLaunchKernelGGL(qk_norm_rope_any_kernel<I8L_BF16>, grid, dim3(256), 0, st, a, interleaved);
    else
      hipLaunchKernelGGL(qk_norm_rope_any_kernel<I8L_F16>, grid, dim3(256), 0, st, a, interleaved);
  }
  return hip_status(hipGetLastError(), "qk_norm_rope launch");
}
