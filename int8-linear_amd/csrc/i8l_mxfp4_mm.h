// Internal interface of the MXFP4 product: its operands, the epilogue and the schedules.
//
//   out[m,n] = cast( sum_b 2^(sa[m,b]+sb[n,b]-254) sum_{i in block b} A[m,i] B[n,i]  (+ bias[n]) )
//
// A [M,K] and B [N,K] hold E2M1 codes, two a byte, sa [M,K/32] and sb [N,K/32] their E8M0 scales;
// the sum is held in fp32 (a block's 32 products are multiples of 1/4 below 2^11: exact), the bias
// is added in fp32 and the result rounded once.
#pragma once

#include "i8l_gemm.h"
#include "i8l_mxfp4.h"

namespace i8l {

struct MxMM {
  const uint8_t *a, *b, *sa, *sb;
  int64_t lda, ldb, ldsa, ldsb;   // bytes from a row to the next
  const void* bias;
  void* out;
  int64_t ldc;                    // elements
  int64_t M, N, K;                // K in elements
  int bias_dtype, out_dtype;
};

__device__ __forceinline__ void mx_store(const MxMM& p, int64_t m, int64_t n, float v) {
  const int64_t at = m * p.ldc + n;
  if (p.out_dtype == I8L_F32) ((float*)p.out)[at] = v;
  else if (p.out_dtype == I8L_BF16) ((uint16_t*)p.out)[at] = f32_to_bf16_bits(v);
  else ((uint16_t*)p.out)[at] = f32_to_f16_bits(v);
}

// Four neighbouring columns n .. n + 3 of row m (n a multiple of 4): the bias, one rounding, one
// store where the columns and the alignment allow it.
__device__ __forceinline__ void mx_store4(const MxMM& p, int64_t m, int64_t n, v4f v) {
  if (n >= p.N) return;
  const int es = p.out_dtype == I8L_F32 ? 4 : 2;
  char* at = (char*)p.out + (m * p.ldc + n) * es;
  if (n + 4 <= p.N) {
    if (p.bias) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += load_bias(p.bias, p.bias_dtype, n + r);
    }
    if (((uintptr_t)at & (4 * es - 1)) == 0) {
      if (p.out_dtype == I8L_F32) *(v4f*)at = v;
      else if (p.out_dtype == I8L_BF16)
        *(uint2*)at = make_uint2(f32x2_to_act2<I8L_BF16>(v[0], v[1]), f32x2_to_act2<I8L_BF16>(v[2], v[3]));
      else
        *(uint2*)at = make_uint2(f32x2_to_act2<I8L_F16>(v[0], v[1]), f32x2_to_act2<I8L_F16>(v[2], v[3]));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) mx_store(p, m, n + r, v[r]);
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < p.N)
      mx_store(p, m, n + r, p.bias ? v[r] + load_bias(p.bias, p.bias_dtype, n + r) : v[r]);
}

// Many tokens (i8l_mxfp4_phased.hip): K in whole pairs of 256-element steps, everything on 16 bytes.
// A workspace lets it split K: its plan never needs more than kMaxParts planes of M x N floats.
bool mx_phased_ok(const MxMM& p);
constexpr int kMaxParts = 8;
struct MxPhasedPlan {
  int tile, splits, bm, bn;   // the tile's index, the parts of K, the tile's rows and columns
};
MxPhasedPlan mx_phased_plan(int64_t M, int64_t N, int64_t K, int64_t workspace);
hipError_t launch_mx_phased(const MxMM& p, void* workspace, int64_t bytes, hipStream_t st);
// Few tokens (i8l_mxfp4_ring.hip): whole 128-element runs of K, rows of codes on 16 bytes and of
// scales on 4.
bool mx_ring_ok(const MxMM& p);
hipError_t launch_mx_ring(const MxMM& p, hipStream_t st);
// Any whole blocks of K (i8l_mxfp4_decode.hip): rows of codes on 16 bytes.
bool mx_decode_ok(const MxMM& p);
hipError_t launch_mx_decode(const MxMM& p, hipStream_t st);

}  // namespace i8l
