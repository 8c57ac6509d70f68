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
// held within [0, R] and to those before them, and a row of A outside [0, M) is read as row 0 or zeros
// and gives NaN, so no content of either reaches out of range.
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
constexpr int64_t kMostColumns = (int64_t)1 << 24;
constexpr int64_t kMostK = (int64_t)1 << 17;   // below it the int32 sum of products of two codes cannot overflow

// The most blocks of `bm` rows that R rows over E experts make.
inline int64_t most_blocks(int64_t R, int64_t E, int bm) {
  const int64_t some = std::min(R, E);             // experts with rows
  return some + (R - some) / bm;
}

// The rows and blocks of 64 experts, one a lane (none past the last expert): an offset counts as the
// largest of those up to it, held within [0, R].  A lane's `upto` is the blocks of its expert and all
// before it; `lowest` and `before` carry from 64 experts to the next, 0 at first.
struct ExpertRows {
  int lo, hi, blocks, upto;
};
__device__ __forceinline__ ExpertRows expert_rows(const Grouped& p, int bm, bool in, int off, int next,
                                                  int& lowest, int& before) {
  ExpertRows x;
  x.lo = wave_max_scan(max(min(max(off, 0), p.R), lowest));
  x.hi = max(min(max(next, 0), p.R), x.lo);
  x.blocks = in ? (x.hi - x.lo + bm - 1) / bm : 0;
  x.upto = before + wave_scan(x.blocks);
  lowest = __builtin_amdgcn_readlane(x.lo, 63);
  before = __builtin_amdgcn_readlane(x.upto, 63);
  return x;
}

// A tile: rows [row0, end) of expert e (up to bm of them), column block `col`.
struct GroupTile {
  int e, row0, end, col;
};

// Tile t of the order expert, column block, row block (so that the row blocks that read the same
// weight rows follow each other); false past the last.  Every lane of a wave calls it with the same
// t and gets the same answer: lane l counts the blocks of experts l, l + 64, ..., 128 at a time (their
// offsets in flight together), until t's is among them.
__device__ __forceinline__ bool find_tile(const Grouped& p, int bm, int cols, int64_t t, GroupTile& g) {
  const int lane = threadIdx.x & 63;
  const int64_t q = t / cols;   // t lies in the expert of block q
  int lowest = 0, before = 0;
  for (int e0 = 0; e0 < p.E; e0 += 128) {
    int off[2], next[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int e = min(e0 + 64 * c + lane, p.E - 1);
      off[c] = p.offsets[e];
      next[c] = p.offsets[e + 1];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const ExpertRows x = expert_rows(p, bm, e0 + 64 * c + lane < p.E, off[c], next[c], lowest, before);
      if (const uint64_t behind = __ballot((int64_t)x.upto > q)) {
        const int owner = __builtin_ctzll(behind);
        const int nb = __builtin_amdgcn_readlane(x.blocks, owner);
        const int first = __builtin_amdgcn_readlane(x.upto, owner) - nb;
        const int local = (int)(t - (int64_t)first * cols);
        g.e = e0 + 64 * c + owner;
        g.col = local / nb;
        g.row0 = __builtin_amdgcn_readlane(x.lo, owner) + local % nb * bm;
        g.end = min(g.row0 + bm, __builtin_amdgcn_readlane(x.hi, owner));
        return true;
      }
    }
  }
  return false;
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
// and far below the output's half step of 2^-9 or 2^-12, and a reciprocal below 2^-126 (a gate under
// -87.3) may be 0; an fp32 output takes the accurate exponential and the division.
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

// ------------------------------------------------------------------ copies into LDS
// What the fast schedules share: buffer loads straight into LDS with the row's byte offset in a
// register and the K position in a scalar.  An offset past the buffer's size reads as zeros, which
// gives rows past the expert's last, whole steps past K and its tail within a step their zeros.
constexpr uint32_t kOutside = 0x80000000u;   // (the buffers are smaller than 2^31 bytes)

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// A buffer of `bytes` bytes from p on, checked byte by byte (raw, no stride).
__device__ __forceinline__ v4u buffer_of(const void* p, uint32_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  return v4u{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
             (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) & 0xffffu,
             (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

// 16 bytes a lane into 1 KiB of LDS from `dst` on.  Assembly, so that the compiler, which cannot count
// these among other requests, places no wait of its own: the schedules' explicit waits cover them.
__device__ __forceinline__ void copy_1k(v4u buf, uint32_t off, int at, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
               ::"v"(off), "s"(buf), "s"(at), "s"(dst) : "memory", "m0");
}
// The same, not kept in the caches (weights that one workgroup reads once).
__device__ __forceinline__ void copy_1k_stream(v4u buf, uint32_t off, int at, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen nt lds"
               ::"v"(off), "s"(buf), "s"(at), "s"(dst) : "memory", "m0");
}

// The scales and bias of 4 neighbouring columns of an expert whose columns start at `at` (past the
// last: the last four's).
struct ColQuad {
  float sb[4], bias[4];
};
template <bool BIAS>
__device__ __forceinline__ ColQuad load_quad(const Grouped& p, int64_t at, int n) {
  n = min(n, p.N - 4);
  ColQuad c;
  const float4 s = *(const float4*)(p.sb + at + n);
  c.sb[0] = s.x, c.sb[1] = s.y, c.sb[2] = s.z, c.sb[3] = s.w;
  if constexpr (BIAS) {
    if (p.bias_dtype == I8L_F32) {
      const float4 b = *(const float4*)((const float*)p.bias + at + n);
      c.bias[0] = b.x, c.bias[1] = b.y, c.bias[2] = b.z, c.bias[3] = b.w;
    } else {
      const uint2 h = *(const uint2*)((const uint16_t*)p.bias + at + n);
      const uint32_t w[4] = {h.x & 0xffffu, h.x >> 16, h.y & 0xffffu, h.y >> 16};
#pragma unroll
      for (int r = 0; r < 4; ++r) c.bias[r] = act_to_f32(w[r], p.bias_dtype);
    }
  }
  return c;
}
template <bool BIAS>
__device__ __forceinline__ float quad_value(int32_t acc, float sa, const ColQuad& c, int r) {
  float v = (float)acc;
  v = v * sa;
  v = v * c.sb[r];
  if constexpr (BIAS) v = v + c.bias[r];
  return v;
}

// Any alignment, any K and N (i8l_grouped_mm.hip).
hipError_t launch_grouped_any(const Grouped& p, hipStream_t st);
// What the two schedules below need of sizes and alignment (i8l_grouped_mm.hip).
bool grouped_fast_ok(const Grouped& p);
// Few rows an expert: 16, 32 or 64 rows x 64 columns (i8l_grouped_ring.hip).
hipError_t launch_grouped_ring(int bm, const Grouped& p, hipStream_t st);
// Macro tiles of bm = 64, 128 or 256 rows x 256 columns (i8l_grouped_phased.hip).  stream (bm up to
// 128): the weights past the caches.
hipError_t launch_grouped_phased(int bm, bool stream, const Grouped& p, hipStream_t st);

}  // namespace i8l
