// The grouped W8A8 product: the kernel for any sizes and alignment, the choice of schedule and the C
// entry point.
#include "i8l_grouped.h"

namespace i8l {

namespace {

// ------------------------------------------------------------------ any sizes and alignment
// 64 rows x 64 columns (with silu: 32 gate columns and their 32 up columns) a workgroup of 4 waves,
// K in steps of 64 bytes through registers into LDS, zeros past K, the rows and the columns; a wave
// multiplies its 16 rows by all columns (v_mfma_i32_16x16x64_i8).  V: the bytes of a load, what the
// operands' alignment allows.
constexpr int kAnyTile = 64, kAnyStep = 64, kAnyPitch = 80;   // (pitch: rows 20 banks apart)

template <int V>
__device__ __forceinline__ v4i load_piece(const int8_t* row, int k, int K, bool in) {
  union {
    v4i q;
    int8_t b[16];
  } u;
  u.q = v4i{};
  if (in) {
#pragma unroll
    for (int i = 0; i < 16; i += V)
      if (k + i < K) __builtin_memcpy(u.b + i, __builtin_assume_aligned(row + k + i, V), V);
  }
  return u.q;
}

template <int V>
__global__ void __launch_bounds__(256) grouped_any(Grouped p, int cols) {
  __shared__ __attribute__((aligned(16))) int8_t sh[2][kAnyTile * kAnyPitch];
  GroupTile g;
  if (!find_tile(p, kAnyTile, cols, (int64_t)blockIdx.y * gridDim.x + blockIdx.x, g)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r16 = lane & 15, quad = lane >> 4;
  const int half = p.N / 2;
  // column x of the tile: a row of B, -1 past the last
  auto column = [&](int x) {
    if (!p.silu) {
      const int n = g.col * kAnyTile + x;
      return n < p.N ? n : -1;
    }
    const int n = g.col * (kAnyTile / 2) + x % (kAnyTile / 2);
    return n < half ? (x < kAnyTile / 2 ? n : half + n) : -1;
  };
  const int lrow = tid >> 2, piece = (tid & 3) * 16;
  const bool ain = g.row0 + lrow < g.end;
  bool ok;
  const int8_t* arow = p.a + (ain ? (int64_t)source_row(p, g.row0 + lrow, ok) * p.lda : 0);
  const int bcol = column(lrow);
  const int8_t* brow = p.b + g.e * p.eb + (int64_t)max(bcol, 0) * p.ldb;
  v4i acc[4] = {};
  for (int k = 0; k < p.K; k += kAnyStep) {
    const v4i av = load_piece<V>(arow, k + piece, p.K, ain);
    const v4i bv = load_piece<V>(brow, k + piece, p.K, bcol >= 0);
    __syncthreads();
    *(v4i*)(sh[0] + lrow * kAnyPitch + piece) = av;
    *(v4i*)(sh[1] + lrow * kAnyPitch + piece) = bv;
    __syncthreads();
    const v4i fa = *(const v4i*)(sh[0] + (16 * wave + r16) * kAnyPitch + 16 * quad);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const v4i fb = *(const v4i*)(sh[1] + (16 * c + r16) * kAnyPitch + 16 * quad);
      acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb, fa, acc[c], 0, 0, 0);
    }
  }
  // a lane holds columns 16 c + 4 quad + r of row 16 wave + r16
  const int i = g.row0 + 16 * wave + r16;
  if (i >= g.end) return;
  const float sam = row_scale(p, i);
  const int64_t at = (int64_t)g.e * p.N;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = column(16 * c + 4 * quad + r);
      if (n < 0) continue;
      const float v = group_value(p, acc[c][r], sam, at + n);
      if (!p.silu) group_store(p, i, n, v);
      else if (c < 2) group_store(p, i, n, group_silu(p, v, group_value(p, acc[c + 2][r], sam, at + half + n)));
    }
}

template <int V>
hipError_t launch_any_v(const Grouped& p, hipStream_t st) {
  const int width = p.silu ? kAnyTile / 2 : kAnyTile;
  const int cols = ((p.silu ? p.N / 2 : p.N) + width - 1) / width;
  // a grid counts 65535 workgroups along y, and its threads below 2^32
  const int64_t tiles = most_blocks(p.R, p.E, kAnyTile) * cols;
  const int64_t gx = std::min<int64_t>(tiles, (int64_t)1 << 20), gy = (tiles + gx - 1) / gx;
  if (gy > 65535) return hipErrorInvalidValue;
  hipLaunchKernelGGL((grouped_any<V>), dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, st, p, cols);
  return hipGetLastError();
}

// The rows of a tile by the rows that an expert has on average (their spread is not known here), where
// one is faster than the next in us, over 2048 -> 1536 and 768 -> 2048 (128 experts), 2048 -> 2816 (60)
// and 4096 -> 28672 (8), random choices, cold weights:
//   ring 16 / 32        at 4 rows 55.1 / 57.9, 39.8 / 37.4, 45.1 / 47.2, 146 / 146; at 8 60.7 / 60.2,
//                       44.5 / 40.8, 51.5 / 51.7, 157 / 150
//   ring 32 / 64        at 8 60.2 / 64.4, 40.8 / 44.3, 51.7 / 53.7, 150 / 150; at 16 73.2 / 74.8,
//                       50.0 / 50.7, 63.7 / 66.3, 165 / 157
//   ring 64 / tile 64   at 16 74.8 / 77.1, 50.7 / 43.9, 66.3 / 68.6, 157 / 202; at 24 87.4 / 87.1,
//                       57.9 / 50.1, 73.5 / 69.4, 167 / 205; at 48 110 / 94.6, 73.4 / 54.7, 90.0 / 76.6,
//                       208 / 206: the ring streams the weights of a long K faster
//   tile 64 / 128       at 48 94.6 / 95.4, 54.7 / 58.7, 76.6 / 74.6, 206 / 211; at 64 93.2 / 92.9,
//                       61.0 / 60.4, 86.9 / 86.1, 209 / 214; at 96 114 / 100, 71.1 / 72.4, 98.2 / 92.5,
//                       237 / 218
//   tile 128 / 256      at 128 116 / 131, 79.1 / 85.2, 94.0 / 101, 242 / 245; at 256 165 / 161,
//                       109 / 114, 145 / 149, 315 / 317; at 512 264 / 245, 176 / 173, 226 / 216, 523 / 517
hipError_t launch_fast(const Grouped& p, hipStream_t st) {
  const int64_t each = p.R / p.E;
  if (each < 6) return launch_grouped_ring(16, p, st);
  if (each < 14) return launch_grouped_ring(32, p, st);
  if (each < (p.K >= 4096 ? 44 : p.K > 1024 ? 20 : 14)) return launch_grouped_ring(64, p, st);
  return launch_grouped_phased(each < 64 ? 64 : each < 256 ? 128 : 256, p, st);
}

}  // namespace

// Offsets of 32 bits with bit 31 to spare, 16-byte pieces of every row, whole vectors of the epilogue.
bool grouped_fast_ok(const Grouped& p) {
  const int es = elt_size(p.out_dtype);
  const int64_t most = (int64_t)kOutside - 1024;   // (a step may be requested past K)
  return p.K % 16 == 0 && aligned16(p.a) && aligned16(p.b) && p.lda % 16 == 0 && p.ldb % 16 == 0 &&
         p.eb % 16 == 0 && p.N % (p.silu ? 16 : 8) == 0 && aligned16(p.sb) && aligned16(p.bias) &&
         aligned16(p.out) && p.ldc * es % 16 == 0 && (int64_t)p.M * p.lda + 2 * p.K < most &&
         (int64_t)p.N * p.ldb + 2 * p.K < most && p.ldc * es < ((int64_t)1 << 22) &&
         (most_blocks(p.R, p.E, 16) + 1) * ((p.N + 31) / 32) < (1 << 22);
}

hipError_t launch_grouped_any(const Grouped& p, hipStream_t st) {
  const uint64_t bits = (uintptr_t)p.a | (uintptr_t)p.b | (uint64_t)p.lda | (uint64_t)p.eb |
                        (uint64_t)p.ldb | (uint64_t)p.K;
  if (bits % 16 == 0) return launch_any_v<16>(p, st);
  if (bits % 8 == 0) return launch_any_v<8>(p, st);
  if (bits % 4 == 0) return launch_any_v<4>(p, st);
  return launch_any_v<1>(p, st);
}

}  // namespace i8l

using namespace i8l;

extern "C" int i8l_w8a8_grouped_mm(const int8_t* a, int64_t lda, int64_t M, const int32_t* rows,
                                   const int8_t* b, int64_t expert_stride, int64_t ldb,
                                   const float* scale_a, int64_t scale_a_len, const float* scale_b,
                                   const void* bias, int32_t bias_dtype, const int32_t* offsets,
                                   void* out, int64_t ldc, int32_t out_dtype, int32_t silu_mul,
                                   int64_t R, int64_t E, int64_t N, int64_t K, void* stream) {
  if (M < 0 || R < 0 || E < 1 || N < 0 || K < 1 || (silu_mul && N % 2) || (R > 0 && !rows && M != R)) {
    set_error("w8a8_grouped_mm: bad sizes M=%lld R=%lld E=%lld N=%lld K=%lld%s", (long long)M,
              (long long)R, (long long)E, (long long)N, (long long)K,
              silu_mul ? " (gate and up halves)" : "");
    return I8L_INVALID_ARG;
  }
  auto float_dt = [](int dt) { return dt == I8L_BF16 || dt == I8L_F16 || dt == I8L_F32; };
  if (!float_dt(out_dtype) || (bias && !float_dt(bias_dtype))) {
    set_error("w8a8_grouped_mm: the output and the bias must be bf16, fp16 or fp32");
    return I8L_UNSUPPORTED;
  }
  if (scale_a_len != 1 && scale_a_len != M) {
    set_error("w8a8_grouped_mm: scale_a has %lld values for %lld rows", (long long)scale_a_len,
              (long long)M);
    return I8L_INVALID_ARG;
  }
  if (E > kMaxExperts || R > kMostRows || M > INT32_MAX || N > ((int64_t)1 << 24) ||
      K >= ((int64_t)1 << 17)) {
    // (the int32 sum of fewer than 2^17 products of two codes cannot overflow)
    set_error("w8a8_grouped_mm: up to %d experts, 2^25 rows, 2^24 columns and a K below 2^17, got "
              "R=%lld E=%lld N=%lld K=%lld", kMaxExperts, (long long)R, (long long)E, (long long)N,
              (long long)K);
    return I8L_UNSUPPORTED;
  }
  if (lda < 0 || ldb < 0 || expert_stride < 0 || (R > 1 && ldc < (silu_mul ? N / 2 : N))) {
    set_error("w8a8_grouped_mm: bad strides (a %lld, b %lld and %lld, out %lld)", (long long)lda,
              (long long)expert_stride, (long long)ldb, (long long)ldc);
    return I8L_INVALID_ARG;
  }
  if (R == 0 || N == 0) return I8L_OK;
  if (M == 0) {
    set_error("w8a8_grouped_mm: %lld rows to read of none", (long long)R);
    return I8L_INVALID_ARG;
  }
  if (!operands_ok("w8a8_grouped_mm", {a, b, scale_a, scale_b, offsets, out})) return I8L_INVALID_ARG;
  Grouped p{a, rows, b, scale_a, scale_b, bias, offsets, out, lda, expert_stride, ldb, ldc};
  p.M = (int)M, p.R = (int)R, p.E = (int)E, p.N = (int)N, p.K = (int)K;
  p.sa_per_row = scale_a_len != 1, p.bias_dtype = bias ? bias_dtype : I8L_DTYPE_NONE;
  p.out_dtype = out_dtype, p.silu = silu_mul != 0;
  const hipStream_t st = (hipStream_t)stream;
  const hipError_t e = grouped_fast_ok(p) ? launch_fast(p, st) : launch_grouped_any(p, st);
  return hip_status(e, "w8a8_grouped_mm launch");
}
