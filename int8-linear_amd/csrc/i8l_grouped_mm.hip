// The grouped W8A8 product: the kernel for any sizes and alignment, the choice of schedule and the C
// entry point.
#include "i8l_grouped.h"

namespace i8l {

namespace {

// ------------------------------------------------------------------ any sizes and alignment
// 64 rows x 64 columns (with silu: 32 gate columns and their 32 up columns) a workgroup of 4 waves,
// K in steps of 64 bytes through registers into LDS, zeros past K, the rows and the columns; a wave
// multiplies its 16 rows by all columns (v_mfma_i32_16x16x64_i8).  V: the bytes of a load, what the
// operands' alignment allows.  Loads, LDS stores and MFMAs follow each other, which is what bounds it:
// with loads of 16 bytes 40 tokens over 128 experts (2048 -> 1536) 75.7 us (the ring 45.6), 4096 over 8
// (4096 -> 28672) 3.0 ms (macro tiles 0.87).
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

// The schedule, by the rows that an expert has on average (their spread is not known here).  Measured in
// us with random choices, some experts taken more than others, and two sets of weights or more in turn,
// past what the Infinity Cache holds.  (At few rows an expert such a choice leaves some without any, whose
// weights are not read: of 128 about 40 at 2 rows, 20 at 4.)  128 experts 2048 -> 1536 / 128 768 -> 2048 /
// 60 2048 -> 2816 / 32 7168 -> 4096 / 8 4096 -> 28672 / 8 14336 -> 4096:
//   ring of 16 rows    at 2 rows 47 / 33 / 41 / 105 / 113 / 61; of 32 49 / 32 / 42 / 104 / 114 / 62
//   ring of 32 rows    at 8 60 / 41 / 52 / 134 / 152 / 74, of 16 61 / 45 / 52 / 144 / 157 / 90, of 64
//                      65 / 44 / 54 / 139 / 151 / 73; at 16 74 / 50 / 64 / 152 / 165 / 96, of 64
//                      75 / 51 / 66 / 148 / 158 / 76
//   tile of 64 rows    at 16 70 / 42 / 64 / 146 / 176 / 100; at 32 79 / 48 / 74 / 182 / 180 / 105,
//                      the ring of 64 95 / 62 / 82 / 178 / 176 / 84: where the tiles fill the card in
//                      whole rounds they stream the weights as fast as the ring and multiply faster
//                      (rounds filled: 1 / 1 / .86 / 1 / .88 / .5)
//   tile of 128 rows   at 32 74 / 47 / 67 / 149 / 180 / 107; at 64 86 / 55 / 80 / 156 / 187 / 117, of 64
//                      88 / 60 / 81 / 178 / 190 / 107
//   weights kept       (tile of 128) at 64 90 / 55 / 82 / 175 / 203 / 123; at 128 105 / 73 / 86 / 205 /
//                      228 / 125, streamed 106 / 74 / 88 / 214 / 235 / 121; at 256 156 / 105 / 139 /
//                      299 / 306 / 211, streamed 163 / 113 / 140 / 330 / 310 / 213
//   tile of 256 rows   at 192 142 / 90 / 116 / 256 / 235 / 155, of 128 132 / 89 / 117 / 282 / 252 / 129;
//                      at 512 237 / 167 / 208 / 495 / 517 / 294, of 128 253 / 174 / 220 / 531 / 516 / 305
struct Schedule {
  int bm;        // rows of a tile
  bool ring;     // tiles of 64 columns, else of 256
  bool stream;   // the weights past the caches
};
// lines: a weight's rows start on cache lines (else two of a row's steps share one).
Schedule schedule_of(int64_t R, int64_t E, int64_t N, int64_t K, bool lines) {
  const int64_t each = R / E;
  // (a ring's grid holds all its tiles, 512 threads each, and counts those below 2^32)
  const bool rings = (most_blocks(R, E, 16) + 32) * ((N + 31) / 32) < (1 << 23) - 32;
  if (each < 6 && rings) return {16, true, true};
  const int64_t tiles = std::min(R, E) * ((N + 255) / 256), cus = cu_count();
  const int64_t room = (tiles + cus - 1) / cus * cus;   // of the rounds that the tiles take
  const int64_t ring = 20 * tiles >= 19 * room ? 10 : 10 * tiles < 7 * room ? 44 : K >= 4096 ? 34 : 18;
  if (each < ring && rings) return {each < 14 ? 32 : 64, true, true};
  if (each < 24) return {64, false, lines};
  if (each < (K > 1024 ? 208 : 400)) return {128, false, lines && each < 112};
  return {256, false, false};
}

hipError_t launch_fast(const Grouped& p, hipStream_t st) {
  const bool lines = ((uintptr_t)p.b | (uint64_t)p.eb | (uint64_t)p.ldb) % 128 == 0;
  const Schedule s = schedule_of(p.R, p.E, p.N, p.K, lines);
  return s.ring ? launch_grouped_ring(s.bm, p, st) : launch_grouped_phased(s.bm, s.stream, p, st);
}

}  // namespace

// Offsets of 32 bits with bit 31 to spare, 16-byte pieces of every row, whole vectors of the epilogue.
// (M counts by itself where A's rows are one row expanded: the row scales lie at 32-bit byte offsets.)
bool grouped_fast_ok(const Grouped& p) {
  const int es = elt_size(p.out_dtype);
  const int64_t most = (int64_t)kOutside - 1024;   // (a step may be requested past K)
  return p.K % 16 == 0 && aligned16(p.a) && aligned16(p.b) && p.lda % 16 == 0 && p.ldb % 16 == 0 &&
         p.eb % 16 == 0 && p.N % (p.silu ? 16 : 8) == 0 && aligned16(p.sb) && aligned16(p.bias) &&
         aligned16(p.out) && p.ldc * es % 16 == 0 && (int64_t)p.M * p.lda + 2 * p.K < most &&
         p.M <= 1 << 30 &&
         (int64_t)p.N * p.ldb + 2 * p.K < most && p.ldc * es < ((int64_t)1 << 22) &&
         (most_blocks(p.R, p.E, 64) + 1) * ((p.N + 127) / 128) < (1 << 30);
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

extern "C" int i8l_w8a8_grouped_mm_tile(int64_t R, int64_t E, int64_t N, int64_t K, int32_t lines,
                                        int32_t* tile_m, int32_t* tile_n, int32_t* streamed) {
  if (!tile_m || !tile_n || !streamed) {
    set_error("w8a8_grouped_mm_tile: an output is NULL");
    return I8L_INVALID_ARG;
  }
  if (R < 0 || E < 1 || N < 0 || K < 1 || E > kMaxExperts || R > kMostRows || N > kMostColumns ||
      K >= kMostK) {
    set_error("w8a8_grouped_mm_tile: bad sizes R=%lld E=%lld N=%lld K=%lld", (long long)R,
              (long long)E, (long long)N, (long long)K);
    return I8L_INVALID_ARG;
  }
  const Schedule s = schedule_of(R, E, N, K, lines != 0);
  *tile_m = s.bm, *tile_n = s.ring ? 64 : 256, *streamed = s.stream;
  return I8L_OK;
}

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
  if (E > kMaxExperts || R > kMostRows || M > INT32_MAX || N > kMostColumns || K >= kMostK) {
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
