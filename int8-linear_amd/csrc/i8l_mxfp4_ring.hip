// MXFP4 product for few tokens: weights streamed once from memory through LDS.
//
// A workgroup covers 16 MT tokens and 16 NT columns; its W waves split K, each taking a run of
// 256-element steps, and their partial sums are added through LDS in wave order.  A wave copies a
// step's rows, 128 bytes of codes each, into its own ring of R buffers with direct-to-LDS loads
// (1 KiB of 8 whole lines an instruction), and 8 steps' scales, 64 bytes a row, at once, so nothing
// but its own vmcnt stands between the copies and its reads.  v_mfma_scale_f32_16x16x128 takes lane
// l's row l % 16; the sum over K may take its blocks in any order, so at substep u lane l holds
// block 2 (l / 16) + u, and both substeps' scales are one 16-bit LDS read, picked by op_sel.  The
// weight is the first operand: a lane's four sums are four neighbouring columns of one token.
//
// What bounds it: HBM for few tokens (4096 -> 28672 at 1 token: 62 MB in 12.5 us, 5.0 TB/s), the
// cache lines a CU takes from L2 for many, which is why NT grows with the tokens and the columns.
// 14336 -> 4096 at 80 tokens: 28 us with the fragments loaded straight into registers (a line a
// lane, as neighbouring lanes hold different rows), 20.7 with each step's 8 bytes of scales copied
// with it (a line a row again), 15.8 so.  Many tokens come here where the macro tiles do not take the
// sizes or the alignment, and read the activations once for every 16 or 32 columns (1792 -> 4096 at 512
// tokens 19.9 us, at 4096 155, 2048 -> 4096 by macro tiles 8.4 and 22.8; 11008 -> 4096 at 4096 500, of
// 11264 84).
#include "i8l_mxfp4_mm.h"

namespace i8l {

namespace {

constexpr int kRow = 128;     // bytes of codes a row and step: 256 elements, 8 blocks
constexpr int kSuper = 8;     // steps whose scales come together: 64 bytes a row

__device__ __forceinline__ v8i mx_widen(v4i a) {
  return __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
}

// Direct-to-LDS loads with a scalar base and a lane's 32-bit offset: 16 (4) bytes a lane, the wave's
// into consecutive LDS from dst on.  As assembly, so that the compiler adds no waits of its own.
__device__ __forceinline__ void copy_16(const uint8_t* base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               ::"v"(off), "s"(base), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void copy_16_nt(const uint8_t* base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
               ::"v"(off), "s"(base), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void copy_4(const uint8_t* base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               ::"v"(off), "s"(base), "s"(dst) : "memory", "m0");
}

// The sizes of a step and of a wave's LDS: HALF has 8 token rows (for up to 8 tokens), not 16.
template <int MT, int NT, bool HALF, int R>
struct RingStep {
  static constexpr int kActRows = HALF ? 8 : 16 * MT;
  static constexpr int kRows = 16 * NT + kActRows;
  static constexpr int kCopies = kRows / 8, kScaleCopies = kRows / 4;
  static constexpr int kStepBytes = kRows * kRow, kScaleBytes = kRows * 8 * kSuper;
  // R steps' codes (weight rows, then token rows), then two batches of scales
  static constexpr int kBytes = R * kStepBytes + 2 * kScaleBytes;
};

template <int MT, int NT, bool HALF, int W, int R>
__global__ void __launch_bounds__(64 * W) mxfp4_ring(MxMM p) {
  typedef RingStep<MT, NT, HALF, R> S;
  static_assert(!HALF || MT == 1, "half a tile of tokens is one tile's");
  static_assert((R - 1) * S::kCopies + S::kScaleCopies < 64, "the copies in flight fit vmcnt");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, row = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
  const int steps = (int)((p.K + 255) / 256), share = (steps + W - 1) / W;
  const int first = wave * share, mine = min(max(steps - first, 0), share);
  const int ragged = p.K % 256 != 0 ? steps - 1 - first : -1;   // the wave's step of half its blocks

  // Lane offsets of the copies.  Copy c of an operand: its rows [8c, 8c + 8), lane l slot l % 8 of
  // row l / 8, which holds chunk (l % 8) ^ (row / 2 % 8); rows past the last copy the last.
  const uint8_t* pb = p.b + n0 * p.ldb + (int64_t)first * kRow;
  const uint8_t* pa = p.a + m0 * p.lda + (int64_t)first * kRow;
  const int last_n = (int)min(p.N - 1 - n0, (int64_t)16 * NT - 1);
  const int last_m = (int)min(p.M - 1 - m0, (int64_t)16 * MT - 1);
  uint32_t off[S::kCopies];
  auto chunk = [&](int r) { return ((lane & 7) ^ ((r >> 1) & 7)) * 16; };
#pragma unroll
  for (int c = 0; c < S::kCopies; ++c) {
    const bool w = c < 2 * NT;
    const int r = 8 * (w ? c : c - 2 * NT) + (lane >> 3);
    off[c] = (uint32_t)(min(r, w ? last_n : last_m) * (int)(w ? p.ldb : p.lda) + chunk(r));
  }
  // Scales: copy c brings 64 bytes of each of rows [4c, 4c + 4) of an operand, lane l slot l % 16 of
  // row l / 16, which holds word (l % 16) ^ 2 (c % 4) (so that the 16 rows of a fragment's read
  // meet different banks).
  const int words = (int)(p.K / 128);   // words of a row's scales
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_i8_t*)lds + wave * S::kBytes;
  auto request_scales = [&](int batch) {
    const uint32_t d = lds0 + R * S::kStepBytes + (batch & 1) * S::kScaleBytes;
    const int w0 = (first + batch * kSuper) * 2;
#pragma unroll
    for (int c = 0; c < S::kScaleCopies; ++c) {
      const bool w = c < 4 * NT;
      const int cc = w ? c : c - 4 * NT;
      const int r = min(4 * cc + (lane >> 4), w ? last_n : last_m);
      const int word = min(w0 + ((lane & 15) ^ ((cc & 3) * 2)), words - 1);
      copy_4(w ? p.sb + n0 * p.ldsb : p.sa + m0 * p.ldsa,
             (uint32_t)(r * (int)(w ? p.ldsb : p.ldsa) + 4 * word), d + c * 256);
    }
  };
  // the copies of the wave's step i; of half a step, the missing chunks copy present ones (not used)
  auto request = [&](int i) {
    if (i % kSuper == 0) request_scales(i / kSuper);
    const uint32_t d = lds0 + (i % R) * S::kStepBytes;
    const int64_t at = (int64_t)i * kRow;
#pragma unroll
    for (int c = 0; c < S::kCopies; ++c) {
      const bool w = c < 2 * NT;
      const int r = 8 * (w ? c : c - 2 * NT) + (lane >> 3);
      const uint32_t o = i == ragged ? off[c] - (chunk(r) & 64) : off[c];
      if (w) copy_16_nt(pb + at, o, d + c * 1024);
      else copy_16(pa + at, o, d + c * 1024);
    }
  };

  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{};

  const uint8_t* mem = lds + wave * S::kBytes;
  const int arow = HALF ? row & 7 : row;
  int fragb[2], fraga[2];   // a row's chunk of substep u: 16-row tiles are 16 * kRow further
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    fragb[u] = row * kRow + (((2 * quarter + u) ^ ((row >> 1) & 7)) * 16);
    fraga[u] = 16 * NT * kRow + arow * kRow + (((2 * quarter + u) ^ ((arow >> 1) & 7)) * 16);
  }
  auto multiply = [&](int i) {
    const uint8_t* d = mem + (i % R) * S::kStepBytes;
    const uint8_t* sc = mem + R * S::kStepBytes + (i / kSuper % 2) * S::kScaleBytes;
    const int word = 2 * (i % kSuper) + (quarter >> 1), odd = 2 * (quarter & 1);
    const uint8_t* scb = sc + row * 64 + (word ^ ((row >> 2) * 2)) * 4 + odd;
    const uint8_t* sca = sc + 16 * NT * 64 + arow * 64 + (word ^ ((arow >> 2) * 2)) * 4 + odd;
    v4i fb[NT][2], fa[MT][2];
    int sb[NT], sa[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      sb[j] = *(const uint16_t*)(scb + j * 16 * 64);
#pragma unroll
      for (int u = 0; u < 2; ++u) fb[j][u] = *(const v4i*)(d + fragb[u] + j * 16 * kRow);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      sa[i] = *(const uint16_t*)(sca + i * 16 * 64);
#pragma unroll
      for (int u = 0; u < 2; ++u) fa[i][u] = *(const v4i*)(d + fraga[u] + i * 16 * kRow);
    }
    if (i == ragged && quarter >= 2) {   // blocks past K: zeros of scale one
#pragma unroll
      for (int j = 0; j < NT; ++j) fb[j][0] = fb[j][1] = v4i{}, sb[j] = 0x7f7f;
#pragma unroll
      for (int i = 0; i < MT; ++i) fa[i][0] = fa[i][1] = v4i{}, sa[i] = 0x7f7f;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            mx_widen(fb[j][0]), mx_widen(fa[i][0]), acc[i][j], 4, 4, 0, sb[j], 0, sa[i]);
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            mx_widen(fb[j][1]), mx_widen(fa[i][1]), acc[i][j], 4, 4, 1, sb[j], 1, sa[i]);
      }
  };

#pragma unroll
  for (int i = 0; i < R - 1; ++i)
    if (i < mine) request(i);
  for (int i = 0; i < mine; ++i) {
    const int ahead = min(R - 1, mine - 1 - i);   // steps in flight behind this one
    if (ahead == R - 1) {
      wait_lgkmcnt0();   // the reads of the buffer to be written have returned
      request(i + R - 1);
    }
    // all but those steps' copies (a batch of scales among them) have landed
    const bool scales = i % kSuper + ahead >= kSuper;
    auto wait = [&](auto n) {
      constexpr int N = decltype(n)::value;
      if (scales) wait_vmcnt_wlds<N * S::kCopies + (N ? S::kScaleCopies : 0)>();
      else wait_vmcnt_wlds<N * S::kCopies>();
    };
    if (R > 3 && ahead == 3) wait(std::integral_constant<int, (R > 3 ? 3 : 0)>{});
    else if (R > 2 && ahead == 2) wait(std::integral_constant<int, (R > 2 ? 2 : 0)>{});
    else if (ahead == 1) wait(std::integral_constant<int, 1>{});
    else wait(std::integral_constant<int, 0>{});
    multiply(i);
  }

  // the waves' sums in wave order, the bias, one rounding: tile x = i NT + j by wave x % W
  __syncthreads();   // every wave's reads and copies are done: the rings become the sums' place
  v4f* part = (v4f*)lds;   // [W][MT NT][64]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[(wave * MT * NT + i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int x = wave; x < MT * NT; x += W) {
    v4f v = part[x * 64 + lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += part[(w * MT * NT + x) * 64 + lane];
    const int64_t m = m0 + 16 * (x / NT) + row, n = n0 + 16 * (x % NT) + 4 * quarter;
    if (m < p.M) mx_store4(p, m, n, v);
  }
}

// Waves and buffers of a variant: four waves of three buffers where the LDS holds them, fewer for
// more rows.  MANY, more than 300 workgroups: two waves, so that a CU holds several workgroups
// (12288 columns at 64 tokens 9.7 -> 7.9 us, 28672 at 16 15.0 -> 13.4).  LONG, few workgroups and a
// long K at up to 16 tokens: eight waves (6144 -> 2048 at 1 token 4.4 -> 4.1 us).
enum Variant { kPlain, kMany, kLong };
template <int ROWS, Variant V>
struct RingShape {
  static constexpr bool fits(int w, int r) {   // the LDS, and vmcnt
    return w * ROWS * 128 * (r + 1) <= (int)kMaxLds && (r - 1) * ROWS / 8 + ROWS / 4 < 64;
  }
  static constexpr int W = V == kLong ? 8 : V == kMany ? 2 : fits(4, 2) ? 4 : fits(3, 2) ? 3 : 2;
  static constexpr int R = V == kMany ? (ROWS <= 64 ? 3 : 2) : fits(W, 3) ? 3 : 2;
};

template <int MT, int NT, bool HALF, Variant V>
hipError_t launch_ring_k(const MxMM& p, hipStream_t st) {
  constexpr int ROWS = 16 * NT + (HALF ? 8 : 16 * MT);
  constexpr int W = RingShape<ROWS, V>::W, R = RingShape<ROWS, V>::R;
  auto kern = mxfp4_ring<MT, NT, HALF, W, R>;
  constexpr size_t shm = std::max<size_t>((size_t)W * RingStep<MT, NT, HALF, R>::kBytes,
                                          (size_t)W * MT * NT * 1024);
  static_assert(shm <= kMaxLds, "the rings fit the LDS");
  static std::atomic<uint64_t> lds_done{0};
  lds_opt_in((const void*)kern, shm, lds_done);
  const dim3 grid((unsigned)((p.N + 16 * NT - 1) / (16 * NT)),
                  (unsigned)((p.M + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL(kern, grid, dim3(64 * W), shm, st, p);
  return hipGetLastError();
}

template <int MT, int NT, bool HALF>
hipError_t launch_ring_v(const MxMM& p, hipStream_t st) {
  const int64_t groups = (p.N + 16 * NT - 1) / (16 * NT) * ((p.M + 16 * MT - 1) / (16 * MT));
  if (groups > 300) return launch_ring_k<MT, NT, HALF, kMany>(p, st);
  if constexpr (MT == 1 && NT == 1)
    if (p.K >= 4096) return launch_ring_k<MT, NT, HALF, kLong>(p, st);
  return launch_ring_k<MT, NT, HALF, kPlain>(p, st);
}

// Columns of a workgroup: 16 where that gives the card few workgroups, more where it has plenty,
// which reads the activations less often; the limits are where the two sides met in sweeps of the
// two models' projections at 1 to 128 tokens (12288 columns at 32 tokens: 16 columns 5.7 us, 64 6.1;
// at 80: 64 columns 9.2, 32 11.1).
template <int MT, bool HALF>
hipError_t launch_ring_n(const MxMM& p, hipStream_t st) {
  const int64_t tiles = (p.N + 15) / 16;
  if (tiles <= 300 || (tiles > 600 && tiles < 1000 && p.M <= 32))
    return launch_ring_v<MT, 1, HALF>(p, st);
  if constexpr (MT <= 6)
    if (tiles >= 600 && (tiles >= 1000 ? p.M > 8 : p.M > 64)) return launch_ring_v<MT, 4, HALF>(p, st);
  return launch_ring_v<MT, 2, HALF>(p, st);
}

}  // namespace

bool mx_ring_ok(const MxMM& p) {
  auto a4 = [](const void* q) { return ((uintptr_t)q & 3) == 0; };
  return aligned16(p.a) && aligned16(p.b) && p.lda % 16 == 0 && p.ldb % 16 == 0 && p.K % 128 == 0 &&
         a4(p.sa) && a4(p.sb) && p.ldsa % 4 == 0 && p.ldsb % 4 == 0 && p.lda <= 1 << 23 &&
         p.ldb <= 1 << 23 && p.ldsa <= 1 << 23 && p.ldsb <= 1 << 23 && (p.M + 127) / 128 <= 65535;
}

hipError_t launch_mx_ring(const MxMM& p, hipStream_t st) {
  if (p.M <= 8) return launch_ring_n<1, true>(p, st);
  switch (std::min<int64_t>((p.M + 15) / 16, 8)) {
    case 1: return launch_ring_n<1, false>(p, st);
    case 2: return launch_ring_n<2, false>(p, st);
    case 3: return launch_ring_n<3, false>(p, st);
    case 4: return launch_ring_n<4, false>(p, st);
    case 5: return launch_ring_n<5, false>(p, st);
    case 6: return launch_ring_n<6, false>(p, st);
  }
  return launch_ring_n<8, false>(p, st);
}

}  // namespace i8l
