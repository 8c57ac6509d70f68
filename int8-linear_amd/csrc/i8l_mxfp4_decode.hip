// MXFP4 product for a K of any whole blocks: operands straight from memory into
// v_mfma_scale_f32_16x16x128.
//
// A workgroup covers 16 MT tokens and 16 NT columns; its W waves take the K steps of 512 elements
// in turn (step s: wave s % W) and their partial sums are added through LDS in wave order.  In a
// step lane l holds row l % 16 of each 16-row tile, block 4 u + l / 16 of its 16 blocks at
// substep u: 16 bytes of codes (16 rows x 64 contiguous bytes an instruction), and byte l / 16 of
// word u of the row's 16 scale bytes, which one load brings.  The weight is the first MFMA operand,
// so a lane's four sums are four neighbouring columns of one token: one store.
//
// What bounds it: cache lines, as the lanes of a load hold 16 different rows: 2752 -> 4096 at 1 token
// 4.2 us, at 64 8.1 (cold weights).  The rows that i8l_mxfp4_ring.hip takes go through LDS instead.
// It is a kernel for few tokens that also takes many, as the macro tiles need whole 512s of K: every
// 16 columns read all activations again (2752 -> 4096 at 512 tokens 41.7 us, at 4096 351; the macro
// tiles at a K of 2560 27 there).
#include "i8l_mxfp4_mm.h"

namespace i8l {

namespace {

constexpr int kStep = 512;   // K elements of a step

__device__ __forceinline__ v8i mx_widen(v4i a) {
  return __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
}

// One 16-row tile's operands of a step.
struct MxFrag {
  v4i c[4];
  uint4 s;
};

// TAIL: the step's blocks past `left` are zeros of scale one.  NT_LOAD: read once, not kept in L2.
template <bool TAIL, bool NT_LOAD>
__device__ __forceinline__ MxFrag load_frag(const uint8_t* q, const uint8_t* s, int quarter,
                                            int left) {
  MxFrag f;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int blk = 4 * u + quarter;
    const v4i* p = (const v4i*)(q + 16 * blk);
    if (TAIL && blk >= left) f.c[u] = v4i{};
    else f.c[u] = NT_LOAD ? __builtin_nontemporal_load(p) : *p;
  }
  if (TAIL) {
    uint32_t w[4] = {0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (4 * u + quarter < left) w[u] = (uint32_t)s[4 * u + quarter] << (8 * quarter);
    f.s = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    __builtin_memcpy(&f.s, s, 16);
  }
  return f;
}

template <int MT, int NT, int W>
__global__ void __launch_bounds__(64 * W) mxfp4_decode(MxMM p) {
  const int lane = threadIdx.x & 63, row = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
  const uint8_t *a[MT], *sa[MT], *b[NT], *sb[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {   // rows past the last read it again and are not stored
    const int64_t m = min(m0 + 16 * i + row, p.M - 1);
    a[i] = p.a + m * p.lda;
    sa[i] = p.sa + m * p.ldsa;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t n = min(n0 + 16 * j + row, p.N - 1);
    b[j] = p.b + n * p.ldb;
    sb[j] = p.sb + n * p.ldsb;
  }
  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{};

  const int steps = (int)(p.K / kStep);
  auto step = [&](auto tail, int t, int left) {
    constexpr bool TAIL = decltype(tail)::value;
    MxFrag fb[NT], fa[MT];
    const int64_t at = (int64_t)t * (kStep / 2), ats = (int64_t)t * (kStep / kMxBlock);
#pragma unroll
    for (int j = 0; j < NT; ++j)
      fb[j] = load_frag<TAIL, true>(b[j] + at, sb[j] + ats, quarter, left);
#pragma unroll
    for (int i = 0; i < MT; ++i)
      fa[i] = load_frag<TAIL, false>(a[i] + at, sa[i] + ats, quarter, left);
    const int sh = 8 * quarter;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      auto word = [&](const MxFrag& f) {
        return (int)((u == 0 ? f.s.x : u == 1 ? f.s.y : u == 2 ? f.s.z : f.s.w) >> sh);
      };
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              mx_widen(fb[j].c[u]), mx_widen(fa[i].c[u]), acc[i][j], 4, 4, 0, word(fb[j]), 0,
              word(fa[i]));
    }
  };
  for (int t = wave; t < steps; t += W) step(std::false_type{}, t, 16);
  if (p.K % kStep && steps % W == wave)
    step(std::true_type{}, steps, (int)(p.K % kStep) / kMxBlock);

  // the waves' sums in wave order, the bias, one rounding: tile x = i NT + j by wave x % W
  extern __shared__ v4f part[];   // [W][MT NT][64]
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

// Tokens of a workgroup: up to 128, in tiles of 16.
constexpr int kMaxMT = 8;

template <int MT, int NT, int W>
hipError_t launch_decode_k(const MxMM& p, hipStream_t st) {
  auto kern = mxfp4_decode<MT, NT, W>;
  constexpr size_t shm = (size_t)W * MT * NT * 1024;
  static_assert(shm <= 64 * 1024, "the partial sums fit the LDS of any launch");
  const dim3 grid((unsigned)((p.N + 16 * NT - 1) / (16 * NT)),
                  (unsigned)((p.M + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL(kern, grid, dim3(64 * W), shm, st, p);
  return hipGetLastError();
}

}  // namespace

bool mx_decode_ok(const MxMM& p) {
  return aligned16(p.a) && aligned16(p.b) && p.lda % 16 == 0 && p.ldb % 16 == 0 &&
         (p.M + 16 * kMaxMT - 1) / (16 * kMaxMT) <= 65535 && p.K <= (int64_t)kStep * INT32_MAX &&
         p.N <= ((int64_t)1 << 27) - 16;   // (512 threads for 16 columns: a grid's stay below 2^32)
}

// Eight waves; the tokens in as few tiles as hold them.
hipError_t launch_mx_decode(const MxMM& p, hipStream_t st) {
  switch (std::min<int64_t>(kMaxMT, (p.M + 15) / 16)) {
    case 1: return launch_decode_k<1, 1, 8>(p, st);
    case 2: return launch_decode_k<2, 1, 8>(p, st);
    case 3:
    case 4: return launch_decode_k<4, 1, 8>(p, st);
  }
  return launch_decode_k<kMaxMT, 1, 8>(p, st);
}

}  // namespace i8l
