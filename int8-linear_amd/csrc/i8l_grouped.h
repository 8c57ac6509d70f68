// Internal interface of the grouped W8A8 product: one int8 weight [N,K] for each expert, the rows
// ordered by expert.
//
//   out[i, n] = cast( f32(sum_k A[r(i), k] * B[e(i), n, k]) * sa[r(i)|0] * sb[e(i), n] (+ bias[e(i), n]) )
//
// Row i belongs to the expert e with offsets[e] <= i < offsets[e + 1] and reads A's row r(i) = rows[i]
// (i itself without `rows`).  The arithmetic is i8l_gemm.h's: exact int32 sums, the epilogue in fp32
// left to right, one cast.  With `silu` the first N / 2 columns are gate values g and the others up
// values u, out [R, N/2] = cast(g / (1 + exp(-g)) * u), g and u in fp32 as the epilogue leaves them.
//
// The offsets are read on the device, so the host knows the rows' number but not their spread: every
// schedule launches for the most row blocks there can be and the workgroups find theirs.  Offsets are
// held within [0, R], an expert's end to its start or behind it, and a row of A outside [0, M) is read
// as row 0 and gives NaN, so no content of either reaches out of range.
#pragma once

#include "i8l_gemm.h"

namespace i8l {

struct Grouped {
  const int8_t* a;
  const int32_t* rows;      // NULL: row i of A
  const int8_t* b;
  const float *sa, *sb;
  const void* bias;
  const int32_t* offsets;   // [E + 1]
  void* out;
  int64_t lda, eb, ldb;     // bytes: A's rows, B's experts, B's rows
  int64_t ldc;              // elements
  int M, R, E, N, K;
  int sa_per_row, bias_dtype, out_dtype, silu;
};

constexpr int kMaxExperts = 512;
constexpr int64_t kMostRows = (int64_t)1 << 25;   // (the sum of any 512 experts' blocks fits an int)

// The most blocks of `bm` rows that R rows over E experts make.
inline int64_t most_blocks(int64_t R, int64_t E, int bm) {
  const int64_t some = std::min(R, E);             // experts with rows
  return some + (R - some) / bm;
}

// Expert e's rows, clamped.
__device__ __forceinline__ void expert_rows(const Grouped& p, int e, int& lo, int& hi) {
  lo = min(max(p.offsets[e], 0), p.R);
  hi = min(max(p.offsets[e + 1], lo), p.R);
}

// A tile: rows [row0, end) of expert e (up to bm of them), column block `col`.
struct GroupTile {
  int e, row0, end, col;
};

// Tile t of the order expert, column block, row block (so that the row blocks that read the same
// weight rows follow each other); false past the last.  Every lane of a wave calls it with the same
// t and gets the same answer: a lane counts the blocks of ceil(E / 64) experts.
__device__ __forceinline__ bool find_tile(const Grouped& p, int bm, int cols, int64_t t, GroupTile& g) {
  const int lane = threadIdx.x & 63, per = (p.E + 63) / 64;
  const int e0 = min(lane * per, p.E), e1 = min(e0 + per, p.E);
  int blocks = 0;
  for (int e = e0; e < e1; ++e) {
    int lo, hi;
    expert_rows(p, e, lo, hi);
    blocks += (hi - lo + bm - 1) / bm;
  }
  const int upto = wave_scan(blocks);
  const int64_t q = t / cols;   // the first block of t's expert is at most this one
  const uint64_t behind = __ballot((int64_t)upto > q);
  if (!behind) return false;
  const int owner = __builtin_ctzll(behind);
  int at = upto - blocks, e = e0, lo = 0, hi = 0, nb = 1;
  for (int x = e0; x < e1; ++x) {
    int l, h;
    expert_rows(p, x, l, h);
    const int b = (h - l + bm - 1) / bm;
    if (at + b > q) {
      e = x, lo = l, hi = h, nb = b;
      break;
    }
    at += b;
  }
  e = __builtin_amdgcn_readlane(e, owner);
  lo = __builtin_amdgcn_readlane(lo, owner);
  hi = __builtin_amdgcn_readlane(hi, owner);
  nb = __builtin_amdgcn_readlane(nb, owner);
  at = __builtin_amdgcn_readlane(at, owner);
  const int64_t local = t - (int64_t)at * cols;
  g.e = e;
  g.col = (int)(local / nb);
  g.row0 = lo + (int)(local % nb) * bm;
  g.end = min(g.row0 + bm, hi);
  return true;
}

// A's row of ordered row i, and its scale: NaN where the row is outside.
__device__ __forceinline__ int source_row(const Grouped& p, int i, bool& ok) {
  const int r = p.rows ? p.rows[i] : i;
  ok = r >= 0 && r < p.M;
  return ok ? r : 0;
}
__device__ __forceinline__ float row_scale(const Grouped& p, int i) {
  bool ok;
  const int r = source_row(p, i, ok);
  const float s = p.sa[p.sa_per_row ? r : 0];
  return ok ? s : __builtin_nanf("");
}

// g / (1 + exp(-g)) * u in fp32.  For a 16-bit output by the hardware's exp2 and reciprocal: the
// rounded argument g * log2(e) makes exp(-g) off by |g| * 2^-24, 2^-17 of it at the end of the range
// and far below the output's half step of 2^-9 or 2^-12; an fp32 output takes the accurate
// exponential and the division.
template <bool F32>
__device__ __forceinline__ float silu_mul(float g, float u) {
  if constexpr (F32) {
    return g / (1.0f + canon_expf(-g)) * u;
  } else {
    const float z = __builtin_amdgcn_exp2f(-1.44269504088896340736f * g);
    return g * __builtin_amdgcn_rcpf(1.0f + z) * u;
  }
}

// One column's epilogue value.
__device__ __forceinline__ float group_value(const Grouped& p, int32_t acc, float sam, int64_t at) {
  float v = (float)acc;
  v = v * sam;
  v = v * p.sb[at];
  if (p.bias) v = v + load_bias(p.bias, p.bias_dtype, at);
  return v;
}

__device__ __forceinline__ void group_store(const Grouped& p, int64_t i, int64_t n, float v) {
  const int64_t at = i * p.ldc + n;
  if (p.out_dtype == I8L_F32) ((float*)p.out)[at] = v;
  else if (p.out_dtype == I8L_BF16) ((uint16_t*)p.out)[at] = f32_to_bf16_bits(v);
  else ((uint16_t*)p.out)[at] = f32_to_f16_bits(v);
}

__device__ __forceinline__ float group_silu(const Grouped& p, float g, float u) {
  return p.out_dtype == I8L_F32 ? silu_mul<true>(g, u) : silu_mul<false>(g, u);
}

// Any alignment, any K and N (i8l_grouped_mm.hip).
hipError_t launch_grouped_any(const Grouped& p, hipStream_t st);
// Macro tiles of bm = 64, 128 or 256 rows x 256 columns (i8l_grouped_phased.hip).
bool grouped_phased_ok(const Grouped& p);
hipError_t launch_grouped_phased(int bm, const Grouped& p, hipStream_t st);

}  // namespace i8l
