// The MXFP4 product: the kernel for any strides and alignment, the choice of schedule and the C
// entry point.
#include "i8l_mxfp4_mm.h"

namespace i8l {

namespace {

// One thread an output, a block of 32 at a time: the block's exact sum, then one scaled addition.
__global__ void __launch_bounds__(256) mxfp4_mm_any(MxMM p) {
  const int64_t n = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int64_t m = (int64_t)blockIdx.y * 4 + (threadIdx.x >> 6);
  if (m >= p.M || n >= p.N) return;
  const uint8_t *a = p.a + m * p.lda, *b = p.b + n * p.ldb;
  const uint8_t *sa = p.sa + m * p.ldsa, *sb = p.sb + n * p.ldsb;
  float acc = 0.0f;
  for (int64_t blk = 0; blk < p.K / kMxBlock; ++blk) {
    float s = 0.0f;
    for (int i = 0; i < kMxBlock / 2; ++i) {
      const uint32_t x = a[blk * 16 + i], y = b[blk * 16 + i];
      s += e2m1_value(x & 15) * e2m1_value(y & 15) + e2m1_value(x >> 4) * e2m1_value(y >> 4);
    }
    const int ea = sa[blk], eb = sb[blk];
    acc += ea == 255 || eb == 255 ? __builtin_nanf("") : __builtin_ldexpf(s, ea + eb - 254);
  }
  if (p.bias) acc += load_bias(p.bias, p.bias_dtype, n);
  mx_store(p, m, n, acc);
}

hipError_t launch_mx_any(const MxMM& p, hipStream_t st) {
  // the grid's y counts up to 65535: longer batches in pieces
  const int64_t most = 65535 * 4;
  for (int64_t m = 0; m < p.M; m += most) {
    MxMM q = p;
    q.M = std::min(most, p.M - m);
    q.a += m * p.lda;
    q.sa += m * p.ldsa;
    q.out = (char*)p.out + m * p.ldc * elt_size(p.out_dtype);
    hipLaunchKernelGGL(mxfp4_mm_any, dim3((unsigned)((p.N + 63) / 64), (unsigned)((q.M + 3) / 4)),
                       dim3(256), 0, st, q);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

// Whether the macro tiles are faster than the ring, by tokens, the more the columns (each in us,
// ring / tiles, cold weights): 28672 columns at 32 tokens 15.1 / 15.9 and at 48 18.5 / 16.5; 12288 at
// 64 7.9 / 8.4 and at 80 9.2 / 8.6; 6144 at 128 11.3 / 14.7; and where a long K is split, 14336 -> 4096
// at 80 15.8 / 16.1 and at 96 18.1 / 16.7 (6144 -> 2048 at 128 11.6 / 12.8).
bool many_tokens(int64_t M, int64_t N, int64_t K, bool split) {
  return M > (N >= 20480 ? 32 : N >= 9216 ? 72 : split && K >= 8192 ? 80 : 128);
}

// Four threads a column (mxfp4_mm_any; the ring's wide launches alike): a grid's stay below 2^32.
constexpr int64_t kMostColumns = ((int64_t)1 << 30) - 64;
constexpr int64_t kMostWorkspace = (int64_t)64 << 20;

// The sizes alone of mx_phased_ok.
bool phased_sizes(int64_t M, int64_t N, int64_t K) {
  return M > 0 && N >= 128 && N % 8 == 0 && K >= 1024 && K % 512 == 0;
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int64_t i8l_mxfp4_mm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (!phased_sizes(M, N, K) || M > 4096 || N > kMostColumns || K > INT32_MAX ||
      !many_tokens(M, N, K, true))
    return 0;
  const int splits = mx_phased_plan(M, N, K, kMostWorkspace).splits;
  return splits > 1 ? splits * M * N * 4 : 0;
}

extern "C" int i8l_mxfp4_mm_tile(int64_t M, int64_t N, int64_t K, int32_t* tile_m, int32_t* tile_n,
                                 int32_t* parts) {
  if (!tile_m || !tile_n || !parts) {
    set_error("mxfp4_mm_tile: an output is NULL");
    return I8L_INVALID_ARG;
  }
  *tile_m = *tile_n = 0;
  *parts = 1;
  const bool split = i8l_mxfp4_mm_workspace_bytes(M, N, K) > 0;
  if (phased_sizes(M, N, K) && M < (int64_t)1 << 30 && N <= kMostColumns && K <= INT32_MAX &&
      many_tokens(M, N, K, split)) {
    const MxPhasedPlan plan = mx_phased_plan(M, N, K, split ? kMostWorkspace : 0);
    *tile_m = plan.bm, *tile_n = plan.bn, *parts = plan.splits;
  }
  return I8L_OK;
}

extern "C" int i8l_mxfp4_mm_ws(const uint8_t* a, int64_t lda, const uint8_t* b, int64_t ldb,
                               const uint8_t* scale_a, int64_t ldsa, const uint8_t* scale_b,
                               int64_t ldsb, const void* bias, int32_t bias_dtype, void* out,
                               int64_t ldc, int32_t out_dtype, int64_t M, int64_t N, int64_t K,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K <= 0 || K % kMxBlock) {
    set_error("mxfp4_mm: bad sizes M=%lld N=%lld K=%lld (K in whole blocks of 32)", (long long)M,
              (long long)N, (long long)K);
    return I8L_INVALID_ARG;
  }
  auto float_dt = [](int dt) { return dt == I8L_BF16 || dt == I8L_F16 || dt == I8L_F32; };
  if (!float_dt(out_dtype) || (bias && !float_dt(bias_dtype))) {
    set_error("mxfp4_mm: the output and the bias must be bf16, fp16 or fp32");
    return I8L_UNSUPPORTED;
  }
  if (M > INT32_MAX || N > kMostColumns || K > INT32_MAX) {
    set_error("mxfp4_mm: M=%lld N=%lld K=%lld: too large", (long long)M, (long long)N, (long long)K);
    return I8L_UNSUPPORTED;
  }
  const int64_t kb = K / 2, ks = K / kMxBlock;
  if ((M > 1 && (lda < kb || ldsa < ks || ldc < N)) || (N > 1 && (ldb < kb || ldsb < ks))) {
    set_error("mxfp4_mm: a row stride is shorter than its row (a %lld, b %lld, scales %lld and "
              "%lld, out %lld for M=%lld N=%lld K=%lld)", (long long)lda, (long long)ldb,
              (long long)ldsa, (long long)ldsb, (long long)ldc, (long long)M, (long long)N,
              (long long)K);
    return I8L_INVALID_ARG;
  }
  if (M == 0 || N == 0) return I8L_OK;
  if (!operands_ok("mxfp4_mm", {a, b, scale_a, scale_b, out})) return I8L_INVALID_ARG;
  const MxMM p{a, b, scale_a, scale_b, lda, ldb, ldsa, ldsb, bias, out, ldc, M, N, K,
               bias ? bias_dtype : I8L_DTYPE_NONE, out_dtype};
  const hipStream_t st = (hipStream_t)stream;
  // a workspace is taken whole or not at all
  const int64_t need = i8l_mxfp4_mm_workspace_bytes(M, N, K);
  const bool split = need > 0 && workspace && workspace_bytes >= need && aligned16(workspace);
  const hipError_t e = mx_phased_ok(p) && (many_tokens(M, N, K, split) || !mx_ring_ok(p))
                           ? launch_mx_phased(p, workspace, split ? kMostWorkspace : 0, st)
                       : mx_ring_ok(p)   ? launch_mx_ring(p, st)
                       : mx_decode_ok(p) ? launch_mx_decode(p, st)
                                         : launch_mx_any(p, st);
  return hip_status(e, "mxfp4_mm launch");
}

extern "C" int i8l_mxfp4_mm(const uint8_t* a, int64_t lda, const uint8_t* b, int64_t ldb,
                            const uint8_t* scale_a, int64_t ldsa, const uint8_t* scale_b,
                            int64_t ldsb, const void* bias, int32_t bias_dtype, void* out,
                            int64_t ldc, int32_t out_dtype, int64_t M, int64_t N, int64_t K,
                            void* stream) {
  return i8l_mxfp4_mm_ws(a, lda, b, ldb, scale_a, ldsa, scale_b, ldsb, bias, bias_dtype, out, ldc,
                         out_dtype, M, N, K, nullptr, 0, stream);
}
