// The grouped W8A8 product for experts with few rows: weights and rows through one ring of LDS slots
// (v_mfma_i32_16x16x64_i8).
#include "i8l_gemm_tile.h"
#include "i8l_grouped.h"

namespace i8l {

namespace {

// ------------------------------------------------------------------ schedule
// A workgroup of 8 waves computes 16 MT rows x 64 columns of one expert (with SILU 32 gate columns and
// their 32 up columns) in 128-byte K steps.  The steps of both operands go through S LDS slots, filled
// S - 1 steps ahead: a slot holds the 64 weight rows and then the 16 MT rows of a step (chunk c of row
// r at slot c ^ (r & 7)).  Wave w multiplies columns 16 (w % 4) .. +15 by every row over half w / 4 of
// each step; the halves' sums meet once, at the end.
//
// What bounds it is the weight stream: a weight byte is copied by one workgroup only (by one for each
// 16 MT rows of its expert), and the slots of two workgroups fill a CU's LDS, so that about 140 KiB are
// in flight a CU and one workgroup's start and end lie under the other's stream.  Sets of weights in turn
// / after a read of 3 GiB: 4 rows of each of 128 experts (2048 -> 1536, 403 MB) 62 / 63 us, 6.5 TB/s;
// 4 tokens through 14 of 60 experts (2048 -> 2816, SILU, 81 MB) 17.2 / 18.0; one token's 8 experts
// (768 -> 2048, 12.6 MB) 5.2 / 6.2.
//
// The start is a chain of dependent reads (offsets, then the rows' indices, then the operands), so the
// weights are requested as soon as the tile is found and the indices come through the scalar cache,
// whose waits do not count the copies; the row scales, which need the indices too, are read at the end.
constexpr int kStep = 128, kCols = 64;
constexpr int kXcdRun = 4;   // tiles in a row for one XCD: an expert's row blocks share its L2

__host__ __device__ constexpr int slots(int mt) { return 80 * 1024 / ((kCols + 16 * mt) * kStep); }

// PLAIN: bf16 output and no bias, at compile time; else what the call says.
template <int MT, bool SILU, bool PLAIN>
__global__ void __launch_bounds__(512) grouped_ring(Grouped p, uint32_t abytes, uint32_t bbytes, int cols) {
  constexpr int W = 8, BM = 16 * MT, BK = kStep;
  constexpr int ROWS = kCols + BM, SLOT = ROWS * BK, S = slots(MT);
  constexpr int WIDE = SILU ? kCols / 2 : kCols;   // output columns
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];

  GroupTile g;
  {
    const int b = blockIdx.x;
    const int t = b / (8 * kXcdRun) * (8 * kXcdRun) + b % 8 * kXcdRun + b / 8 % kXcdRun;
    if (!find_tile(p, BM, cols, t, g)) return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, grp = lane >> 4;
  const int cg = wave & 3, kh = wave >> 2;
  const int width = SILU ? p.N / 2 : p.N;
  const int ns = (p.K + BK - 1) / BK;

  // Copies: wave w brings weight rows 8 w .. +7 of a step and, for w < 2 MT, rows 8 w .. +7 of A;
  // lane l fetches chunk (l % 8) ^ (row & 7) of row l / 8.
  const int l8 = lane >> 3, chunk = ((lane & 7) ^ l8) * 16;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_i8*)lds + wave * 1024;
  const v4u bufB = buffer_of(p.b + g.e * p.eb, bbytes);
  const v4u bufA = buffer_of(p.a, abytes);
  // (eight columns: all within the problem or all past it, then the last eight again, not stored)
  const int x = 8 * wave;
  const int brow = SILU ? (x < WIDE ? min(g.col * WIDE + x, width - 8)
                                    : width + min(g.col * WIDE + x - WIDE, width - 8))
                        : min(g.col * WIDE + x, width - 8);
  const uint32_t voffB = (uint32_t)(l8 * (int)p.ldb + chunk);
  const int bat = brow * (int)p.ldb;
  auto outside = [&](int t) { return t * BK + chunk < p.K ? 0u : kOutside; };
  auto requestB = [&](int t, int slot) {
    copy_1k_stream(bufB, voffB | outside(t), bat + t * BK, lds0 + slot * SLOT);
  };
  const bool hasA = wave < 2 * MT;
  uint32_t voffA = kOutside;
  auto requestA = [&](int t, int slot) {
    if (hasA) copy_1k(bufA, voffA | outside(t), t * BK, lds0 + slot * SLOT + kCols * BK);
  };
  auto request = [&](int t, int slot) {
    requestB(t, slot);
    requestA(t, slot);
  };
  // the rows of this lane's outputs, for their scales (used at the end), and this wave's eight rows of A
  int src[MT], at[8];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = min(g.row0 + 16 * i + r16, p.R - 1);
    src[i] = p.rows ? p.rows[r] : r;
  }
  if (hasA) {
    typedef const __attribute__((address_space(4))) int32_t scalar_i32;
    scalar_i32* rows = (scalar_i32*)(uintptr_t)p.rows;
#pragma unroll
    for (int j = 0; j < 8; ++j) at[j] = min(g.row0 + x + j, p.R - 1);
    if (p.rows) {
#pragma unroll
      for (int j = 0; j < 8; ++j) at[j] = rows[at[j]];
    }
  }
#pragma unroll
  for (int t = 0; t < S - 1; ++t)
    if (t < ns) requestB(t, t);
  if (hasA) {
    int r = at[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) r = l8 == j ? at[j] : r;
    voffA = g.row0 + x + l8 < g.end && r >= 0 && r < p.M ? (uint32_t)(r * (int)p.lda + chunk) : kOutside;
#pragma unroll
    for (int t = 0; t < S - 1; ++t)
      if (t < ns) requestA(t, t);
  }

  const int bofs = (16 * cg + r16) * BK + (((4 * kh + grp) ^ (r16 & 7)) * 16);
  const int aofs = (kCols + r16) * BK + (((4 * kh + grp) ^ (r16 & 7)) * 16);
  v4i acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = v4i{0, 0, 0, 0};
  auto multiply = [&](int slot) {
    const int8_t* base = lds + slot * SLOT;
    const v4i b = *(const v4i*)(base + bofs);
    v4i a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) a[i] = *(const v4i*)(base + aofs + i * 16 * BK);
    __builtin_amdgcn_sched_barrier(0);   // every read in flight before the first MFMA waits
#pragma unroll
    for (int i = 0; i < MT; ++i)
      acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, a[i], acc[i], 0, 0, 0);
  };
  // Step t: its copies have landed everywhere and every wave is done with step t - 1, whose slot
  // then takes step t + S - 1.  What a wave has requested behind step t's copies: S - 2 steps of B, and
  // where it brings A too, whose first S - 1 steps stand behind B's, S - 2 + t copies up to t = S - 2
  // and twice S - 2 from there on.
  auto landed = [&](int t) {
    if (!hasA) {
      wait_vmcnt_lgkm0<S - 2>();
      return;
    }
    switch (t) {
      case 0: wait_vmcnt_lgkm0<S - 2>(); break;
      case 1: wait_vmcnt_lgkm0<S - 1>(); break;
      case 2: wait_vmcnt_lgkm0<S>(); break;
      case 3: wait_vmcnt_lgkm0<std::min(S + 1, 2 * S - 4)>(); break;
      case 4: wait_vmcnt_lgkm0<std::min(S + 2, 2 * S - 4)>(); break;
      case 5: wait_vmcnt_lgkm0<std::min(S + 3, 2 * S - 4)>(); break;
      default: wait_vmcnt_lgkm0<2 * S - 4>();
    }
  };
  static_assert(S >= 4 && S <= 8, "the cases above");
  int t = 0, slot = 0;
  for (; t + S - 1 < ns; ++t) {
    landed(t);
    lds_barrier();
    request(t + S - 1, slot == 0 ? S - 1 : slot - 1);
    multiply(slot);
    slot = slot + 1 == S ? 0 : slot + 1;
  }
  // The last S - 1 steps (fewer on a short K): at least one copy for each step behind t is requested
  // behind its copies; the waits are coarser, for half of them and then for all.
  constexpr int H = (S - 1) / 2;
  for (; t < ns; ++t) {
    if (ns - 1 - t >= H) wait_vmcnt_lgkm0<H>();
    else wait_vmcnt_lgkm0<0>();
    lds_barrier();
    multiply(slot);
    slot = slot + 1 == S ? 0 : slot + 1;
  }
  float sam[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const bool ok = src[i] >= 0 && src[i] < p.M;
    const float s = p.sa[p.sa_per_row && ok ? src[i] : 0];
    sam[i] = ok ? s : __builtin_nanf("");
  }

  // the other half's sums (and with SILU the up columns') through LDS to the waves that store
  constexpr int STORE = SILU ? 2 : 4;
  __syncthreads();
  v4i* red = (v4i*)lds;   // [8][MT][64]
  if (wave >= STORE) {
#pragma unroll
    for (int i = 0; i < MT; ++i) red[(wave * MT + i) * 64 + lane] = acc[i];
  }
  __syncthreads();
  if (wave >= STORE) return;
  const int n = g.col * WIDE + 16 * cg + 4 * grp;
  if (n >= width) return;
  const int64_t ecol = (int64_t)g.e * p.N;
  auto finish = [&](auto biased, auto store) {
    constexpr bool BIAS = decltype(biased)::value;
    const ColQuad cl = load_quad<BIAS>(p, ecol, n);
    const ColQuad cu = load_quad<BIAS>(p, ecol, SILU ? width + n : n);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int row = g.row0 + 16 * i + r16;
      const v4i sum = acc[i] + red[((wave + 4) * MT + i) * 64 + lane];
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = quad_value<BIAS>(sum[r], sam[i], cl, r);
      if constexpr (SILU) {
        const v4i up = red[((wave + 2) * MT + i) * 64 + lane] + red[((wave + 6) * MT + i) * 64 + lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float u = quad_value<BIAS>(up[r], sam[i], cu, r);
          v[r] = PLAIN ? silu_mul<false>(v[r], u) : group_silu(p, v[r], u);
        }
      }
      if (row < g.end) store(row, v);
    }
  };
  auto store16 = [&](int row, const float (&v)[4]) {
    uint2 h;
    if (PLAIN || p.out_dtype == I8L_BF16)
      h = make_uint2(f32x2_to_act2<I8L_BF16>(v[0], v[1]), f32x2_to_act2<I8L_BF16>(v[2], v[3]));
    else
      h = make_uint2(f32x2_to_act2<I8L_F16>(v[0], v[1]), f32x2_to_act2<I8L_F16>(v[2], v[3]));
    *(uint2*)((uint16_t*)p.out + (int64_t)row * p.ldc + n) = h;
  };
  if constexpr (PLAIN) {
    finish(std::false_type{}, store16);
  } else {
    auto any = [&](int row, const float (&v)[4]) {
      if (p.out_dtype == I8L_F32)
        *(float4*)((float*)p.out + (int64_t)row * p.ldc + n) = make_float4(v[0], v[1], v[2], v[3]);
      else
        store16(row, v);
    };
    if (p.bias) finish(std::true_type{}, any);
    else finish(std::false_type{}, any);
  }
}

// ------------------------------------------------------------------ host side
template <int MT, bool SILU, bool PLAIN>
hipError_t launch_k(const Grouped& p, hipStream_t st) {
  auto kern = grouped_ring<MT, SILU, PLAIN>;
  constexpr size_t shm = (size_t)slots(MT) * (kCols + 16 * MT) * kStep;
  static_assert(8 * MT * 1024 <= shm, "the sums fit the ring");
  static std::atomic<uint64_t> lds_done{0};  // devices this kernel is opted in on
  lds_opt_in((const void*)kern, shm, lds_done);
  const int width = SILU ? p.N / 2 : p.N, wide = SILU ? kCols / 2 : kCols;
  const int cols = (width + wide - 1) / wide;
  constexpr int round = 8 * kXcdRun;
  const int64_t tiles = (most_blocks(p.R, p.E, 16 * MT) * cols + round - 1) / round * round;
  const uint32_t abytes = (uint32_t)((int64_t)(p.M - 1) * p.lda + p.K);
  const uint32_t bbytes = (uint32_t)((int64_t)(p.N - 1) * p.ldb + p.K);
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(512), shm, st, p, abytes, bbytes, cols);
  return hipGetLastError();
}

template <int MT>
hipError_t launch_t(const Grouped& p, hipStream_t st) {
  const bool plain = p.out_dtype == I8L_BF16 && !p.bias;
  if (p.silu) return plain ? launch_k<MT, true, true>(p, st) : launch_k<MT, true, false>(p, st);
  return plain ? launch_k<MT, false, true>(p, st) : launch_k<MT, false, false>(p, st);
}

}  // namespace

hipError_t launch_grouped_ring(int bm, const Grouped& p, hipStream_t st) {
  if (bm == 16) return launch_t<1>(p, st);
  if (bm == 32) return launch_t<2>(p, st);
  return launch_t<4>(p, st);
}

}  // namespace i8l
