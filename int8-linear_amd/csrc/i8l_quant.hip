// Fused per-token int8 quantizers for MI355X (gfx950): add+RMSNorm+quantize,
// SiLU-and-mul+quantize and the plain per-token quantizer.
//
// Arithmetic follows the reference's Triton kernels step for step
// (AshrithaG/int8-linear, int8_linear/fused_quant.py): the residual add and the norm in
// fp32 (60-69), the normalized value rounded to the weight dtype, multiplied by the weight
// and rounded to the activation dtype (72), the SiLU and its rounding (84-87), and the
// quantizer _quantize_row (41-53):
//     scale = absmax / 127;  inv = absmax == 0 ? 0 : 127 / absmax;
//     q = clamp(rne(y * inv), -128, 127)
// Three points the reference leaves to Triton/libdevice are fixed here so that the CPU
// oracle reproduces every bit:
//   * sum(x^2) is a pairwise tree in double over the row padded with zeros to a power of
//     two, leaf i = x_i^2 (exact in double);  var = f32(sum / H);
//   * rsqrt(v) = f32(1 / sqrt(double(v))) (IEEE double sqrt and divide);
//   * exp is canon_expf (Cody-Waite + degree-7 Taylor with explicit fma).
// Compiled with -ffp-contract=off: every other operation is the single IEEE fp32 op written.
//
// Launch layout.  A token row is owned by NW waves (NW = 1 for rows up to 2048 elements),
// and a workgroup holds RPB rows.  The row is cut into 8-element chunks; lane l of wave w
// owns chunks (w*J + j)*64 + l for j < J, so each load instruction of a wave reads 64
// consecutive chunks (1 KiB of bf16) and each lane's chunk j is an aligned 8-leaf subtree.
// The sum of squares is then evaluated as the perfect binary tree over the padded row:
// the 8 leaves of a chunk in-lane, 64 chunks by a lane butterfly (DPP within 16-lane rows,
// a swizzle across rows, a readlane across the halves) into an aligned 512-element node,
// the J nodes of a wave pairwise, and the NW waves pairwise through LDS.  IEEE addition is
// commutative, so both partners of each butterfly step hold the same node.  Maxima are
// order-free.  A row owned by one wave needs no LDS and no barrier.
#include "i8l_quant_row.h"

namespace i8l {

namespace {

// The quantizer of a row whose values y (J chunks of 8 per lane) are final: absmax over the
// row, scale and reciprocal, codes stored as 8-byte pieces, the scale by the row's first lane.
template <int J, bool VEC, bool MULTI, bool FULL = false>
__device__ __forceinline__ void quantize_store(float (&y)[J][8], const RowPos& p, int n, int nw,
                                               int8_t* qrow, float* scale_out, int precise,
                                               float* sh) {
  float am = 0.0f;
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) am = fmaxf(am, fabsf(y[j][i]));
  const float absmax = row_max<MULTI>(am, p, nw, sh);
  // both division conventions, selected (once per row: no branch on the path)
  const float s_div = absmax / 127.0f;
  const float i_div = absmax == 0.0f ? 0.0f : 127.0f / absmax;
  const float s_rcp = absmax * (1.0f / 127.0f);
  const float i_rcp = absmax == 0.0f ? 0.0f : 127.0f * (1.0f / absmax);
  const float scale = precise ? s_div : s_rcp;
  const float inv = precise ? i_div : i_rcp;
  if (p.rw == 0 && p.lane == 0) *scale_out = scale;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e0 = chunk_base<J>(p, j);
    if (VEC) {
      if (FULL || e0 < n) {
        const float* v = y[j];
        *(uint2*)(qrow + e0) =
            make_uint2(code_rne4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                       code_rne4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e0 + i < n) qrow[e0 + i] = (int8_t)code_rne(y[j][i] * inv);
    }
  }
}

// ------------------------------------------------------------------ add + RMSNorm + quant
template <int J, int DT, int WDT, bool VEC, bool RES, bool MULTI, bool FULL>
__global__ void __launch_bounds__(1024)
add_rmsnorm_quant_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ res,
                         const uint16_t* __restrict__ w, float eps, int8_t* __restrict__ q,
                         float* __restrict__ scale, uint16_t* __restrict__ rout, int64_t M,
                         int H, int nw, int rpb, int precise) {
  pin_vals(x, res, w, eps, q, scale, rout, M, H, nw, rpb, precise);
  __shared__ double dsh[kMaxWaves];
  __shared__ float fsh[kMaxWaves];
  const RowPos p = row_pos<MULTI>(nw, rpb);
  if (p.row >= M) return;  // whole single-wave rows only: a row of nw > 1 waves has rpb = 1
  const int64_t ro = p.row * H;
  float xv[J][8];
  norm_row<J, DT, WDT, VEC, RES, MULTI, FULL>(x, res, w, eps, rout, ro, H, nw, p, dsh, xv);
  quantize_store<J, VEC, MULTI, FULL>(xv, p, H, nw, q + ro, scale + p.row, precise, fsh);
}

// ------------------------------------------------------------------ SiLU-and-mul + quant
// FULL (row length exactly NW*J*512): no bounds checks.
template <int J, int DT, bool VEC, bool ROUND, bool MULTI, bool FULL>
__global__ void __launch_bounds__(1024)
silu_mul_quant_kernel(const uint16_t* __restrict__ gu, int8_t* __restrict__ q,
                      float* __restrict__ scale, int64_t M, int I, int nw, int rpb,
                      int precise) {
  pin_vals(gu, q, scale, M, I, nw, rpb, precise);
  __shared__ float fsh[kMaxWaves];
  const RowPos p = row_pos<MULTI>(nw, rpb);
  if (p.row >= M) return;
  float y[J][8];
  silu_row<J, DT, VEC, ROUND, FULL>(gu + p.row * 2 * I, I, p, y);
  quantize_store<J, VEC, MULTI, FULL>(y, p, I, nw, q + p.row * I, scale + p.row, precise, fsh);
}

// ------------------------------------------------------------------ plain per-token quant
template <int J, int DT, bool VEC, bool MULTI, bool FULL>
__global__ void __launch_bounds__(1024)
quant_kernel(const uint16_t* __restrict__ x, int64_t ldx, int8_t* __restrict__ q,
             float* __restrict__ scale, int64_t M, int H, int nw, int rpb, int precise) {
  pin_vals(x, ldx, q, scale, M, H, nw, rpb, precise);
  __shared__ float fsh[kMaxWaves];
  const RowPos p = row_pos<MULTI>(nw, rpb);
  if (p.row >= M) return;
  float y[J][8];
#pragma unroll
  for (int j = 0; j < J; ++j) load8<DT, VEC, FULL>(x + p.row * ldx, chunk_base<J>(p, j), H, y[j]);
  quantize_store<J, VEC, MULTI, FULL>(y, p, H, nw, q + p.row * H, scale + p.row, precise, fsh);
}

// Kernel selection: the element path (VEC false) is built for J = 4 only.  The residual and
// the multi-wave row are compile-time choices of the kernel, not branches inside it.
template <int DT, int WDT, bool RES, bool MULTI>
void launch_norm_k(const Geom& g, bool vec, dim3 grid, hipStream_t st, const uint16_t* x,
                   const uint16_t* res, const uint16_t* w, float eps, int8_t* q, float* scale,
                   uint16_t* rout, int64_t M, int H, int precise) {
#define I8L_NORM(J_, V_, F_)                                                                \
  hipLaunchKernelGGL((add_rmsnorm_quant_kernel<J_, DT, WDT, V_, RES, MULTI, F_>), grid,      \
                     block_of(g), 0, st, x, res, w, eps, q, scale, rout, M, H, g.nw, g.rpb,   \
                     precise)
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
void launch_norm(const Geom& g, bool vec, dim3 grid, hipStream_t st, const uint16_t* x,
                 const uint16_t* res, const uint16_t* w, float eps, int8_t* q, float* scale,
                 uint16_t* rout, int64_t M, int H, int precise) {
  const bool multi = g.nw > 1;
  if (res)
    multi ? launch_norm_k<DT, WDT, true, true>(g, vec, grid, st, x, res, w, eps, q, scale, rout, M, H, precise)
          : launch_norm_k<DT, WDT, true, false>(g, vec, grid, st, x, res, w, eps, q, scale, rout, M, H, precise);
  else
    multi ? launch_norm_k<DT, WDT, false, true>(g, vec, grid, st, x, res, w, eps, q, scale, rout, M, H, precise)
          : launch_norm_k<DT, WDT, false, false>(g, vec, grid, st, x, res, w, eps, q, scale, rout, M, H, precise);
}

template <int DT, bool ROUND, bool MULTI>
void launch_silu_k(const Geom& g, bool vec, dim3 grid, hipStream_t st, const uint16_t* gu,
                   int8_t* q, float* scale, int64_t M, int I, int precise) {
#define I8L_SILU(J_, V_, F_)                                                                \
  hipLaunchKernelGGL((silu_mul_quant_kernel<J_, DT, V_, ROUND, MULTI, F_>), grid, block_of(g), \
                     0, st, gu, q, scale, M, I, g.nw, g.rpb, precise)
  const bool full = vec && I == 512 * g.j * g.nw;
  if (!vec) I8L_SILU(4, false, false);
  else if (g.j == 1 && full) I8L_SILU(1, true, true);
  else if (g.j == 1) I8L_SILU(1, true, false);
  else if (g.j == 2 && full) I8L_SILU(2, true, true);
  else if (g.j == 2) I8L_SILU(2, true, false);
  else if (g.j == 3) I8L_SILU(3, true, false);
  else if (full) I8L_SILU(4, true, true);
  else I8L_SILU(4, true, false);
#undef I8L_SILU
}

template <int DT, bool ROUND>
void launch_silu(const Geom& g, bool vec, dim3 grid, hipStream_t st, const uint16_t* gu,
                 int8_t* q, float* scale, int64_t M, int I, int precise) {
  if (g.nw > 1)
    launch_silu_k<DT, ROUND, true>(g, vec, grid, st, gu, q, scale, M, I, precise);
  else
    launch_silu_k<DT, ROUND, false>(g, vec, grid, st, gu, q, scale, M, I, precise);
}

template <int DT, bool MULTI>
void launch_quant_k(const Geom& g, bool vec, dim3 grid, hipStream_t st, const uint16_t* x,
                    int64_t ldx, int8_t* q, float* scale, int64_t M, int H, int precise) {
#define I8L_QUANT(J_, V_, F_)                                                               \
  hipLaunchKernelGGL((quant_kernel<J_, DT, V_, MULTI, F_>), grid, block_of(g), 0, st, x, ldx, \
                     q, scale, M, H, g.nw, g.rpb, precise)
  const bool full = vec && H == 512 * g.j * g.nw;
  if (!vec) I8L_QUANT(4, false, false);
  else if (g.j == 1) I8L_QUANT(1, true, false);
  else if (g.j == 2) I8L_QUANT(2, true, false);
  else if (g.j == 3) I8L_QUANT(3, true, false);
  else if (full) I8L_QUANT(4, true, true);
  else I8L_QUANT(4, true, false);
#undef I8L_QUANT
}

template <int DT>
void launch_quant(const Geom& g, bool vec, dim3 grid, hipStream_t st, const uint16_t* x,
                  int64_t ldx, int8_t* q, float* scale, int64_t M, int H, int precise) {
  if (g.nw > 1)
    launch_quant_k<DT, true>(g, vec, grid, st, x, ldx, q, scale, M, H, precise);
  else
    launch_quant_k<DT, false>(g, vec, grid, st, x, ldx, q, scale, M, H, precise);
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int i8l_add_rmsnorm_quant(const void* x, const void* residual, const void* weight,
                                     float eps, int8_t* q, float* scale, void* residual_out,
                                     int64_t M, int64_t H, int32_t act_dtype, int32_t w_dtype,
                                     int32_t precise_div, void* stream) {
  if (M < 0 || H <= 0) {
    set_error("add_rmsnorm_quant: bad sizes M=%lld H=%lld", (long long)M, (long long)H);
    return I8L_INVALID_ARG;
  }
  if (!act_ok(act_dtype) || !act_ok(w_dtype)) {
    set_error("add_rmsnorm_quant: activations and weight must be bf16 or fp16");
    return I8L_UNSUPPORTED;
  }
  if ((residual == nullptr) != (residual_out == nullptr)) {
    set_error("add_rmsnorm_quant: residual and residual_out must both be given or both NULL");
    return I8L_INVALID_ARG;
  }
  if (H > 32768 || M > INT32_MAX) {
    set_error("add_rmsnorm_quant: rows longer than 32768 or more than 2^31 rows");
    return I8L_UNSUPPORTED;
  }
  if (M == 0) return I8L_OK;
  if (!operands_ok("add_rmsnorm_quant", {x, weight, q, scale})) return I8L_INVALID_ARG;
  const int h = (int)H;
  const bool vec = h % 8 == 0 && a16(x) && a16(weight) && a16(q) &&
                   (!residual || (a16(residual) && a16(residual_out)));
  const Geom g = norm_geom(M, h, vec);
  const hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto launch) {
    launch(g, vec, grid_of(M, g), st, (const uint16_t*)x, (const uint16_t*)residual,
           (const uint16_t*)weight, eps, q, scale, (uint16_t*)residual_out, M, h, precise_div);
  };
  if (act_dtype == I8L_BF16)
    w_dtype == I8L_BF16 ? go(launch_norm<I8L_BF16, I8L_BF16>) : go(launch_norm<I8L_BF16, I8L_F16>);
  else
    w_dtype == I8L_BF16 ? go(launch_norm<I8L_F16, I8L_BF16>) : go(launch_norm<I8L_F16, I8L_F16>);
  return hip_status(hipGetLastError(), "add_rmsnorm_quant launch");
}

extern "C" int i8l_silu_mul_quant(const void* gate_up, int8_t* q, float* scale, int64_t M,
                                  int64_t I, int32_t act_dtype, int32_t round_silu,
                                  int32_t precise_div, void* stream) {
  if (M < 0 || I <= 0) {
    set_error("silu_mul_quant: bad sizes M=%lld I=%lld", (long long)M, (long long)I);
    return I8L_INVALID_ARG;
  }
  if (!act_ok(act_dtype)) {
    set_error("silu_mul_quant: activations must be bf16 or fp16");
    return I8L_UNSUPPORTED;
  }
  if (I > 32768 || M > INT32_MAX) {
    set_error("silu_mul_quant: rows longer than 32768 or more than 2^31 rows");
    return I8L_UNSUPPORTED;
  }
  if (M == 0) return I8L_OK;
  if (!operands_ok("silu_mul_quant", {gate_up, q, scale})) return I8L_INVALID_ARG;
  const int i = (int)I;
  const bool vec = i % 8 == 0 && a16(gate_up) && a16(q);
  const hipStream_t st = (hipStream_t)stream;
  const Geom g = silu_geom(M, i, vec);
  auto go = [&](auto launch) {
    launch(g, vec, grid_of(M, g), st, (const uint16_t*)gate_up, q, scale, M, i, precise_div);
  };
  if (act_dtype == I8L_BF16)
    round_silu ? go(launch_silu<I8L_BF16, true>) : go(launch_silu<I8L_BF16, false>);
  else
    round_silu ? go(launch_silu<I8L_F16, true>) : go(launch_silu<I8L_F16, false>);
  return hip_status(hipGetLastError(), "silu_mul_quant launch");
}

extern "C" int i8l_quant_per_token(const void* x, int64_t ldx, int8_t* q, float* scale,
                                   int64_t M, int64_t H, int32_t act_dtype, int32_t precise_div,
                                   void* stream) {
  if (M < 0 || H <= 0 || ldx < H) {
    set_error("quant_per_token: bad sizes M=%lld H=%lld ldx=%lld", (long long)M, (long long)H,
              (long long)ldx);
    return I8L_INVALID_ARG;
  }
  if (!act_ok(act_dtype)) {
    set_error("quant_per_token: activations must be bf16 or fp16");
    return I8L_UNSUPPORTED;
  }
  if (H > 32768 || M > INT32_MAX) {
    set_error("quant_per_token: rows longer than 32768 or more than 2^31 rows");
    return I8L_UNSUPPORTED;
  }
  if (M == 0) return I8L_OK;
  if (!operands_ok("quant_per_token", {x, q, scale})) return I8L_INVALID_ARG;
  const int h = (int)H;
  const bool vec = h % 8 == 0 && ldx % 8 == 0 && a16(x) && a16(q);
  const Geom g = flat_geom(M, h, vec);
  const hipStream_t st = (hipStream_t)stream;
  if (act_dtype == I8L_BF16)
    launch_quant<I8L_BF16>(g, vec, grid_of(M, g), st, (const uint16_t*)x, ldx, q, scale, M, h,
                           precise_div);
  else
    launch_quant<I8L_F16>(g, vec, grid_of(M, g), st, (const uint16_t*)x, ldx, q, scale, M, h,
                          precise_div);
  return hip_status(hipGetLastError(), "quant_per_token launch");
}
