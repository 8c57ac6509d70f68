// MXFP4 quantizers for MI355X (gfx950): the plain one and its inverse, add+RMSNorm+quantize and
// SiLU-and-mul+quantize.
//
//   code_b = E8M0 of max_i |x_i| over a block of 32,   q_i = e2m1(x_i / 2^(code_b - 127))
//
// (i8l_mxfp4.h: the scale rule and the roundings).  The norm and the SiLU-and-mul are those of
// the int8 quantizers (i8l_quant_row.h), the SiLU rounded to the activation dtype as the served
// models compute it, so the values that are quantized are theirs bit for bit.
//
// What bounds them: HBM (reading 2 bytes and writing 17/32 of one an element).  A lane takes
// 8 consecutive elements (16 bytes of bf16 or fp16) and a quad a block, whose maximum is two
// lane moves; each load of a wave reads 1 KiB and each store of codes writes 256 bytes.  No block
// crosses a wave, so nothing is exchanged through LDS except the norm's sum of squares.
#include "i8l_mxfp4.h"
#include "i8l_quant_row.h"

namespace i8l {

namespace {

// The scale bytes of a wave's J chunks: lane l stores chunk l % 4's for its quad (chunk j holds
// blocks 16 j .. 16 j + 15 of the wave's), so four chunks leave in one 64-byte store.
// srow: the row's scales; e0: the wave's first element of the row; n: the row's length.
template <int J>
__device__ __forceinline__ void store_scales(const uint32_t (&code)[J], uint8_t* srow, int64_t e0,
                                             int64_t n, int lane) {
  // the bytes of one word, picked by a shift (a choice among the array's elements goes through LDS,
  // addressed by the block size, which is read from the dispatch packet in host memory: +13 us)
  uint32_t w = code[0];
#pragma unroll
  for (int i = 1; i < J; ++i) w |= code[i] << (8 * i);
  const int j = lane & 3;
  const int64_t e = e0 + (int64_t)(j * 64 + (lane & 60)) * 8;
  if (j < J && e < n) srow[e / kMxBlock] = (uint8_t)(w >> (8 * j));
}

// One word of codes to q (element e0 of a row of n); VEC: q is 4-byte aligned.
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* q, uint32_t w) {
  if (VEC) {
    *(uint32_t*)q = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = (uint8_t)(w >> (8 * i));
  }
}

// Blocks quantized from a lane's J chunks of floats (the fused kernels).
template <int J, bool VEC, bool FULL>
__device__ __forceinline__ void mx_quantize_store(const float (&y)[J][8], const RowPos& p, int n,
                                                  uint8_t* qrow, uint8_t* srow, int rounded) {
  uint32_t code[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    uint32_t am = 0;   // magnitudes as bits: a NaN is above every number
#pragma unroll
    for (int i = 0; i < 8; ++i) am = max(am, __float_as_uint(y[j][i]) & 0x7fffffffu);
    code[j] = mx_scale_code(quad_max(am), rounded);
    const int e0 = chunk_base<J>(p, j);
    if (FULL || e0 < n) store_codes<VEC>(qrow + e0 / 2, mx_codes8(y[j], code[j]));
  }
  store_scales<J>(code, srow, (int64_t)p.rw * J * 512, n, p.lane);
}

// ------------------------------------------------------------------ add + RMSNorm + quant
template <int J, int DT, int WDT, bool VEC, bool RES, bool MULTI, bool FULL>
__global__ void __launch_bounds__(1024)
add_rmsnorm_mxfp4_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ res,
                         const uint16_t* __restrict__ w, float eps, uint8_t* __restrict__ q,
                         uint8_t* __restrict__ scale, uint16_t* __restrict__ rout, int64_t M, int H,
                         int nw, int rpb, int rounded) {
  pin_vals(x, res, w, eps, q, scale, rout, M, H, nw, rpb, rounded);
  __shared__ double dsh[kMaxWaves];
  const RowPos p = row_pos<MULTI>(nw, rpb);
  if (p.row >= M) return;  // whole single-wave rows only: a row of nw > 1 waves has rpb = 1
  const int64_t ro = p.row * H;
  float y[J][8];
  norm_row<J, DT, WDT, VEC, RES, MULTI, FULL>(x, res, w, eps, rout, ro, H, nw, p, dsh, y);
  mx_quantize_store<J, VEC, FULL>(y, p, H, q + ro / 2, scale + ro / kMxBlock, rounded);
}

// ------------------------------------------------------------------ SiLU-and-mul + quant
// A wave's work: J * 512 elements of a row, piece `wave % per_row` of row `wave / per_row`.
template <int J, int DT, bool VEC, bool FULL>
__global__ void __launch_bounds__(256)
silu_mul_mxfp4_kernel(const uint16_t* __restrict__ gu, uint8_t* __restrict__ q,
                      uint8_t* __restrict__ scale, uint32_t waves, uint32_t per_row, int I,
                      int rounded) {
  pin_vals(gu, q, scale, waves, per_row, I, rounded);
  const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave >= waves) return;
  RowPos p;
  p.row = wave / per_row;
  p.rw = wave % per_row;
  p.lane = threadIdx.x & 63;
  p.slot = 0;
  float y[J][8];
  silu_row<J, DT, VEC, true, FULL>(gu + p.row * 2 * I, I, p, y);
  mx_quantize_store<J, VEC, FULL>(y, p, I, q + p.row * (I / 2), scale + p.row * (I / kMxBlock),
                                  rounded);
}

// ------------------------------------------------------------------ plain quantizer
// The same pieces of rows, from memory: K elements a row, ldx apart (contiguous rows come as one).
template <int J, int DT, bool VEC>
__global__ void __launch_bounds__(256)
mxfp4_quant_kernel(const void* __restrict__ xv, int64_t ldx, uint8_t* __restrict__ q,
                   uint8_t* __restrict__ scale, uint32_t waves, uint32_t per_row, int64_t K,
                   int rounded) {
  pin_vals(xv, ldx, q, scale, waves, per_row, K, rounded);
  const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave >= waves) return;
  const int lane = threadIdx.x & 63;
  const int64_t row = wave / per_row;
  const int64_t e0 = (int64_t)(wave % per_row) * (J * 512);
  uint8_t* qrow = q + row * (K / 2);
  uint32_t code[J];
  if constexpr (DT == I8L_F32) {
    const float* x = (const float*)xv + row * ldx;
    float y[J][8];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t e = e0 + (j * 64 + lane) * 8;
      const bool in = e < K;
      if constexpr (VEC) {
        const float4 a = in ? *(const float4*)(x + e) : make_float4(0, 0, 0, 0);
        const float4 b = in ? *(const float4*)(x + e + 4) : make_float4(0, 0, 0, 0);
        y[j][0] = a.x, y[j][1] = a.y, y[j][2] = a.z, y[j][3] = a.w;
        y[j][4] = b.x, y[j][5] = b.y, y[j][6] = b.z, y[j][7] = b.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[j][i] = in ? x[e + i] : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t e = e0 + (j * 64 + lane) * 8;
      uint32_t am = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) am = max(am, __float_as_uint(y[j][i]) & 0x7fffffffu);
      code[j] = mx_scale_code(quad_max(am), rounded);
      if (e < K) store_codes<VEC>(qrow + e / 2, mx_codes8(y[j], code[j]));
    }
  } else {
    const uint16_t* x = (const uint16_t*)xv + row * ldx;
    uint4 v[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t e = e0 + (j * 64 + lane) * 8;
      v[j] = make_uint4(0, 0, 0, 0);
      if (e < K) v[j] = VEC ? *(const uint4*)(x + e) : load_raw8<false>(x + e, 0, 8);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t e = e0 + (j * 64 + lane) * 8;
      typedef unsigned short v2u __attribute__((ext_vector_type(2)));
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
      v2u m = {0, 0};   // magnitudes as bits, two at a time
#pragma unroll
      for (int i = 0; i < 4; ++i)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(v2u, w[i] & 0x7fff7fffu));
      const uint32_t am = quad_max(max((uint32_t)m[0], (uint32_t)m[1]));
      code[j] = mx_scale_code(__float_as_uint(act_to_f32<DT>(am)), rounded);
      if (e < K) store_codes<VEC>(qrow + e / 2, mx_codes8<DT>(v[j], code[j]));
    }
  }
  store_scales<J>(code, scale + row * (K / kMxBlock), e0, K, lane);
}

// ------------------------------------------------------------------ dequantizer
// Values of the same pieces: a lane's word of codes becomes 8 elements.  Every product is exact in
// float and bf16 (two bits times a power of two, subnormals too); fp16 rounds past its range.
template <int J, int OD, bool VEC>
__global__ void __launch_bounds__(256)
mxfp4_dequant_kernel(const uint8_t* __restrict__ q, int64_t ldq, const uint8_t* __restrict__ scale,
                     int64_t lds, void* __restrict__ out, uint32_t waves, uint32_t per_row,
                     int64_t K) {
  pin_vals(q, ldq, scale, lds, out, waves, per_row, K);
  const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave >= waves) return;
  const int lane = threadIdx.x & 63;
  const int64_t row = wave / per_row;
  const int64_t e0 = (int64_t)(wave % per_row) * (J * 512);
  const uint8_t* qrow = q + row * ldq;
  const uint8_t* srow = scale + row * lds;
  uint32_t w[J], code[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int64_t e = e0 + (j * 64 + lane) * 8;
    w[j] = 0, code[j] = 127;
    if (e < K) {
      if constexpr (VEC) {
        w[j] = *(const uint32_t*)(qrow + e / 2);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[j] |= (uint32_t)qrow[e / 2 + i] << (8 * i);
      }
      code[j] = srow[e / kMxBlock];
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int64_t e = e0 + (j * 64 + lane) * 8;
    if (e >= K) continue;
    // 2^(code - 127) for the conversions, which take its exponent field; NaN blocks are set after
    const float s = __uint_as_float(code[j] == 255u ? 0u : code[j] << 23);
    const bool nan = code[j] == 255u;
    float f[8];
#define I8L_FP4_PAIR(i)                                                             \
  {                                                                                 \
    const v2f t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], s, i);             \
    f[2 * i] = nan ? __builtin_nanf("") : t.x;                                      \
    f[2 * i + 1] = nan ? __builtin_nanf("") : t.y;                                  \
  }
    I8L_FP4_PAIR(0) I8L_FP4_PAIR(1) I8L_FP4_PAIR(2) I8L_FP4_PAIR(3)
#undef I8L_FP4_PAIR
    const int64_t at = row * K + e;
    if constexpr (OD == I8L_F32) {
      float4* o = (float4*)((float*)out + at);
      o[0] = make_float4(f[0], f[1], f[2], f[3]);
      o[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      *(uint4*)((uint16_t*)out + at) =
          make_uint4(f32x2_to_act2<OD>(f[0], f[1]), f32x2_to_act2<OD>(f[2], f[3]),
                     f32x2_to_act2<OD>(f[4], f[5]), f32x2_to_act2<OD>(f[6], f[7]));
    }
  }
}

// ------------------------------------------------------------------ host side
// Chunks a lane takes: one while the launch has at most kSpreadWaves waves (a short launch is
// latency-bound), else four, which keeps 4 KiB of a wave's loads in flight.
int chunks_of(int64_t rows, int64_t n) {
  return rows * ((n + 511) / 512) <= kSpreadWaves ? 1 : 4;
}

bool a4(const void* p) { return ((uintptr_t)p & 3) == 0; }

// Waves of a launch whose waves take j chunks of 512 elements of a row each.
int64_t waves_of(int64_t rows, int64_t n, int j) { return rows * ((n + 512 * j - 1) / (512 * j)); }

// Checks shared by the entry points: whole blocks, sizes that the grids can count.
int mx_sizes(const char* who, int64_t M, int64_t K, int64_t most) {
  if (M < 0 || K <= 0 || K % kMxBlock) {
    set_error("%s: rows of %lld values (%lld of them): whole blocks of 32 are needed", who,
              (long long)K, (long long)M);
    return I8L_INVALID_ARG;
  }
  if (K > most || M > INT32_MAX || M * ((K + 511) / 512) > INT32_MAX) {
    set_error("%s: %lld rows of %lld values: too large", who, (long long)M, (long long)K);
    return I8L_UNSUPPORTED;
  }
  return I8L_OK;
}

template <int DT, int WDT, bool RES, bool MULTI>
void launch_mx_norm_k(const Geom& g, bool vec, hipStream_t st, const uint16_t* x,
                      const uint16_t* res, const uint16_t* w, float eps, uint8_t* q, uint8_t* scale,
                      uint16_t* rout, int64_t M, int H, int rounded) {
#define I8L_NORM(J_, V_, F_)                                                                  \
  hipLaunchKernelGGL((add_rmsnorm_mxfp4_kernel<J_, DT, WDT, V_, RES, MULTI, F_>),             \
                     grid_of(M, g), block_of(g), 0, st, x, res, w, eps, q, scale, rout, M, H,  \
                     g.nw, g.rpb, rounded)
  const bool full = vec && H == 512 * g.j * g.nw;
  if (!vec) I8L_NORM(4, false, false);
  else if (g.j == 1 && full) I8L_NORM(1, true, true);
  else if (g.j == 1) I8L_NORM(1, true, false);
  else if (g.j == 2 && full) I8L_NORM(2, true, true);
  else if (g.j == 2) I8L_NORM(2, true, false);
  else if (full) I8L_NORM(4, true, true);
  else I8L_NORM(4, true, false);
#undef I8L_NORM
}

template <int DT, int WDT>
void launch_mx_norm(const Geom& g, bool vec, hipStream_t st, const uint16_t* x, const uint16_t* res,
                    const uint16_t* w, float eps, uint8_t* q, uint8_t* scale, uint16_t* rout,
                    int64_t M, int H, int rounded) {
  const bool multi = g.nw > 1;
  auto go = [&](auto resc, auto multic) {
    launch_mx_norm_k<DT, WDT, decltype(resc)::value, decltype(multic)::value>(
        g, vec, st, x, res, w, eps, q, scale, rout, M, H, rounded);
  };
  if (res) multi ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
  else multi ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
}

template <int DT>
void launch_mx_silu(int j, bool vec, hipStream_t st, const uint16_t* gu, uint8_t* q, uint8_t* scale,
                    int64_t M, int I, int rounded) {
  const uint32_t per_row = (uint32_t)((I + 512 * j - 1) / (512 * j));
  const uint32_t waves = (uint32_t)(M * per_row);
  const bool full = vec && I % (512 * j) == 0;
#define I8L_SILU(J_, V_, F_)                                                                \
  hipLaunchKernelGGL((silu_mul_mxfp4_kernel<J_, DT, V_, F_>), dim3((waves + 3) / 4), dim3(256), \
                     0, st, gu, q, scale, waves, per_row, I, rounded)
  if (!vec) I8L_SILU(1, false, false);
  else if (j == 1 && full) I8L_SILU(1, true, true);
  else if (j == 1) I8L_SILU(1, true, false);
  else if (full) I8L_SILU(2, true, true);
  else I8L_SILU(2, true, false);
#undef I8L_SILU
}

template <int DT>
void launch_mx_quant(int j, bool vec, hipStream_t st, const void* x, int64_t ldx, uint8_t* q,
                     uint8_t* scale, int64_t rows, int64_t K, int rounded) {
  const uint32_t per_row = (uint32_t)((K + 512 * j - 1) / (512 * j));
  const uint32_t waves = (uint32_t)(rows * per_row);
#define I8L_QUANT(J_, V_)                                                                \
  hipLaunchKernelGGL((mxfp4_quant_kernel<J_, DT, V_>), dim3((waves + 3) / 4), dim3(256), 0, \
                     st, x, ldx, q, scale, waves, per_row, K, rounded)
  if (!vec) I8L_QUANT(1, false);
  else if (j == 1) I8L_QUANT(1, true);
  else I8L_QUANT(4, true);
#undef I8L_QUANT
}

template <int OD>
void launch_mx_dequant(int j, bool vec, hipStream_t st, const uint8_t* q, int64_t ldq,
                       const uint8_t* scale, int64_t lds, void* out, int64_t rows, int64_t K) {
  const uint32_t per_row = (uint32_t)((K + 512 * j - 1) / (512 * j));
  const uint32_t waves = (uint32_t)(rows * per_row);
#define I8L_DEQUANT(J_, V_)                                                                  \
  hipLaunchKernelGGL((mxfp4_dequant_kernel<J_, OD, V_>), dim3((waves + 3) / 4), dim3(256), 0, \
                     st, q, ldq, scale, lds, out, waves, per_row, K)
  if (!vec) I8L_DEQUANT(1, false);
  else if (j == 1) I8L_DEQUANT(1, true);
  else I8L_DEQUANT(4, true);
#undef I8L_DEQUANT
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int i8l_mxfp4_quant(const void* x, int64_t ldx, uint8_t* q, uint8_t* scale, int64_t M,
                               int64_t K, int32_t x_dtype, int32_t round_scale, void* stream) {
  if (const int st = mx_sizes("mxfp4_quant", M, K, INT32_MAX)) return st;
  if (ldx < K) {
    set_error("mxfp4_quant: a row stride of %lld for rows of %lld", (long long)ldx, (long long)K);
    return I8L_INVALID_ARG;
  }
  if (!act_ok(x_dtype) && x_dtype != I8L_F32) {
    set_error("mxfp4_quant: values must be bf16, fp16 or fp32");
    return I8L_UNSUPPORTED;
  }
  if (M == 0) return I8L_OK;
  if (!operands_ok("mxfp4_quant", {x, q, scale})) return I8L_INVALID_ARG;
  const int64_t elt = x_dtype == I8L_F32 ? 4 : 2;
  const bool vec = a16(x) && ldx * elt % 16 == 0 && a4(q);
  const bool one = ldx == K;   // rows that touch are one long row of whole blocks
  const int64_t rows = one ? 1 : M, n = one ? M * K : K;
  const int j = vec ? chunks_of(rows, n) : 1;
  if (!waves_ok("mxfp4_quant", waves_of(rows, n, j))) return I8L_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  switch (x_dtype) {
    case I8L_BF16: launch_mx_quant<I8L_BF16>(j, vec, st, x, ldx, q, scale, rows, n, round_scale); break;
    case I8L_F16: launch_mx_quant<I8L_F16>(j, vec, st, x, ldx, q, scale, rows, n, round_scale); break;
    default: launch_mx_quant<I8L_F32>(j, vec, st, x, ldx, q, scale, rows, n, round_scale);
  }
  return hip_status(hipGetLastError(), "mxfp4_quant launch");
}

extern "C" int i8l_mxfp4_dequant(const uint8_t* q, int64_t ldq, const uint8_t* scale, int64_t lds,
                                 void* out, int64_t M, int64_t K, int32_t out_dtype, void* stream) {
  if (const int st = mx_sizes("mxfp4_dequant", M, K, INT32_MAX)) return st;
  if (M > 1 && (ldq < K / 2 || lds < K / kMxBlock)) {
    set_error("mxfp4_dequant: row strides of %lld and %lld for rows of %lld", (long long)ldq,
              (long long)lds, (long long)K);
    return I8L_INVALID_ARG;
  }
  if (!act_ok(out_dtype) && out_dtype != I8L_F32) {
    set_error("mxfp4_dequant: values must be bf16, fp16 or fp32");
    return I8L_UNSUPPORTED;
  }
  if (M == 0) return I8L_OK;
  if (!operands_ok("mxfp4_dequant", {q, scale, out})) return I8L_INVALID_ARG;
  if (!a16(out)) {
    set_error("mxfp4_dequant: the output must be 16-byte aligned");
    return I8L_UNSUPPORTED;
  }
  const bool one = ldq == K / 2 && lds == K / kMxBlock;
  const bool vec = a4(q) && (one || M == 1 || ldq % 4 == 0);
  const int64_t rows = one ? 1 : M, n = one ? M * K : K;
  const int j = vec ? chunks_of(rows, n) : 1;
  if (!waves_ok("mxfp4_dequant", waves_of(rows, n, j))) return I8L_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  switch (out_dtype) {
    case I8L_BF16: launch_mx_dequant<I8L_BF16>(j, vec, st, q, ldq, scale, lds, out, rows, n); break;
    case I8L_F16: launch_mx_dequant<I8L_F16>(j, vec, st, q, ldq, scale, lds, out, rows, n); break;
    default: launch_mx_dequant<I8L_F32>(j, vec, st, q, ldq, scale, lds, out, rows, n);
  }
  return hip_status(hipGetLastError(), "mxfp4_dequant launch");
}

extern "C" int i8l_add_rmsnorm_mxfp4_quant(const void* x, const void* residual, const void* weight,
                                           float eps, uint8_t* q, uint8_t* scale,
                                           void* residual_out, int64_t M, int64_t H,
                                           int32_t act_dtype, int32_t w_dtype, int32_t round_scale,
                                           void* stream) {
  if (const int st = mx_sizes("add_rmsnorm_mxfp4_quant", M, H, 32768)) return st;
  if (!act_ok(act_dtype) || !act_ok(w_dtype)) {
    set_error("add_rmsnorm_mxfp4_quant: activations and weight must be bf16 or fp16");
    return I8L_UNSUPPORTED;
  }
  if ((residual == nullptr) != (residual_out == nullptr)) {
    set_error("add_rmsnorm_mxfp4_quant: residual and residual_out must both be given or both NULL");
    return I8L_INVALID_ARG;
  }
  if (M == 0) return I8L_OK;
  if (!operands_ok("add_rmsnorm_mxfp4_quant", {x, weight, q, scale})) return I8L_INVALID_ARG;
  const int h = (int)H;
  const bool vec = a16(x) && a16(weight) && a4(q) &&
                   (!residual || (a16(residual) && a16(residual_out)));
  const Geom g = norm_geom(M, h, vec);
  if (!waves_ok("add_rmsnorm_mxfp4_quant", M * g.nw)) return I8L_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto launch) {
    launch(g, vec, st, (const uint16_t*)x, (const uint16_t*)residual, (const uint16_t*)weight, eps,
           q, scale, (uint16_t*)residual_out, M, h, round_scale);
  };
  if (act_dtype == I8L_BF16)
    w_dtype == I8L_BF16 ? go(launch_mx_norm<I8L_BF16, I8L_BF16>)
                        : go(launch_mx_norm<I8L_BF16, I8L_F16>);
  else
    w_dtype == I8L_BF16 ? go(launch_mx_norm<I8L_F16, I8L_BF16>)
                        : go(launch_mx_norm<I8L_F16, I8L_F16>);
  return hip_status(hipGetLastError(), "add_rmsnorm_mxfp4_quant launch");
}

extern "C" int i8l_silu_mul_mxfp4_quant(const void* gate_up, uint8_t* q, uint8_t* scale, int64_t M,
                                        int64_t I, int32_t act_dtype, int32_t round_scale,
                                        void* stream) {
  if (const int st = mx_sizes("silu_mul_mxfp4_quant", M, I, 1 << 24)) return st;
  if (!act_ok(act_dtype)) {
    set_error("silu_mul_mxfp4_quant: activations must be bf16 or fp16");
    return I8L_UNSUPPORTED;
  }
  if (M == 0) return I8L_OK;
  if (!operands_ok("silu_mul_mxfp4_quant", {gate_up, q, scale})) return I8L_INVALID_ARG;
  const int i = (int)I;
  const bool vec = a16(gate_up) && a4(q);
  const int j = vec && M * ((I + 511) / 512) > kSiluWaves ? 2 : 1;
  if (!waves_ok("silu_mul_mxfp4_quant", waves_of(M, I, j))) return I8L_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  if (act_dtype == I8L_BF16)
    launch_mx_silu<I8L_BF16>(j, vec, st, (const uint16_t*)gate_up, q, scale, M, i, round_scale);
  else
    launch_mx_silu<I8L_F16>(j, vec, st, (const uint16_t*)gate_up, q, scale, M, i, round_scale);
  return hip_status(hipGetLastError(), "silu_mul_mxfp4_quant launch");
}
