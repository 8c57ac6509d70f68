// MXFP4 product for many tokens: the phased schedule of i8l_gemm_phased.hip with
// v_mfma_scale_f32_32x32x64_f8f6f4 and the scales' own way through LDS.
//
// Persistent BM x BN tiles by 4 waves (2 x 2); a K step is 256 elements, 128 bytes of codes a row,
// cut into four phases, one a quadrant of a wave's tile, whose reads and copies are those of the
// int8 schedule: phase 0 multiplies (A0, Bf), reads Bs(t), requests A0(t+2); 1: (A0, Bs), A1(t),
// Bf(t+2); 2: (A1, Bs), A0(t+1), Bs(t+2); 3: (A1, Bf), the next phase 0's B, A1(t+2), with
// f = t % 2, s = 1 - f, and each phase ends when its wave's reads are back and all but the newest
// five halves have landed, with one workgroup barrier.
//
// A lane holds row l % 32 of a fragment and, as the sum over K may take its blocks in any order,
// blocks 4 (l / 32) .. + 3 of the step's 8 at substeps 0 .. 3: the four scales are one word of the
// row's 8 bytes, picked by op_sel.  The scales of two steps (16 bytes a row of A and B) are one
// batch, in two buffers; a batch is requested at the start of phase 0 of an even step, two steps
// before its first use, by then older than the half that phase 1 of the next step awaits.
//
// What bounds it: MFMA at the clock its power leaves.  On random operands v_mfma alone reaches 6.4 to
// 6.7 PFLOP/s (9.9 on zeros); here the MFMAs are busy 60% of the time at 1.76 GHz (68% within a
// tile's steps, the rest its epilogue): 4096 -> 28672 at 4096 tokens 215 to 227 us, 4.2 to 4.5 PFLOP/s (236 with
// cold weights), 1.4 to 1.5 times what the instruction alone would take, 14336 -> 4096 103 us, 4.7.
#include "i8l_gemm_tile.h"
#include "i8l_mxfp4_mm.h"

namespace i8l {

namespace {

__device__ __forceinline__ void copy_1k(const uint8_t* base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               ::"v"(off), "s"(base), "s"(dst) : "memory", "m0");
}

__device__ __forceinline__ v8i mx_widen(v4i a) {
  return __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
}

// One MFMA with the scales of substep kk, byte kk of each word (op_sel is an immediate).
__device__ __forceinline__ v16f mx_mfma(v4i b, v4i a, v16f c, int sb, int sa, int kk) {
  const v8i x = mx_widen(b), y = mx_widen(a);
  switch (kk) {
    case 0: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, 0, sb, 0, sa);
    case 1: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, 1, sb, 1, sa);
    case 2: return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, 2, sb, 2, sa);
  }
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, 3, sb, 3, sa);
}

// The bias of columns n .. n + 3 (n a multiple of 4, an aligned bias), as floats.
__device__ __forceinline__ void bias4(const MxMM& p, int64_t n, float (&b)[4]) {
  if (p.bias_dtype == I8L_F32) {
    const float4 v = *(const float4*)((const float*)p.bias + n);
    b[0] = v.x, b[1] = v.y, b[2] = v.z, b[3] = v.w;
  } else {
    const uint2 v = *(const uint2*)((const uint16_t*)p.bias + n);
    const uint32_t w[4] = {v.x & 0xffffu, v.x >> 16, v.y & 0xffffu, v.y >> 16};
#pragma unroll
    for (int r = 0; r < 4; ++r) b[r] = act_to_f32(w[r], p.bias_dtype);
  }
}

// SPLIT: K in `splits` parts, each a tile's work of its own, whose fp32 sums go to a plane of M x N
// of p.out each (OD fp32, no bias).
template <int QA, int QB0, int QB1, int OD, bool BIAS, bool SPLIT>
__global__ void __launch_bounds__(256) mxfp4_phased(MxMM p, int group_m, int tiles, int splits) {
  static_assert(!SPLIT || (OD == I8L_F32 && !BIAS), "parts are raw sums");
  constexpr int W = 4, WN = 2, BK = 128;
  constexpr int QB[2] = {QB0, QB1};
  constexpr int QN = QB0 + QB1;                      // column fragments of a wave
  constexpr int BM = 128 * QA, BN = 64 * QN;
  constexpr int CPR = BK / 16, RPC = 64 / CPR;       // chunks of a row, rows of a copy
  constexpr int KK = BK / 32;                        // MFMA substeps of a step
  constexpr int HA = BM / 2 * BK;                    // bytes of an A half
  constexpr int HB[2] = {64 * QB0 * BK, 64 * QB1 * BK};
  constexpr int JA = HA / 1024 / W, JB[2] = {HB[0] / 1024 / W, HB[1] / 1024 / W};  // copies a wave
  constexpr int SC = (BM + BN) / 64;                 // copies of a batch of scales
  constexpr int JS = (SC + W - 1) / W;               // ... a wave (the odd ones are copied twice)
  constexpr int B0 = 4 * HA;                         // LDS: A [buffer][half], B, scales, staging
  constexpr int SB = HB[0] + HB[1];
  constexpr int SC0 = B0 + 2 * SB, SCB = (BM + BN) * 16;
  constexpr int STG = SC0 + 2 * SCB;
  static_assert(QB1 <= QB0 && QB1 >= 1, "the first B half is the larger");
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];

  const int M = (int)p.M, N = (int)p.N;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int num_pid_m = (M + BM - 1) / BM, num_pid_n = (N + BN - 1) / BN;
  const int pairs = (int)(p.K / (4 * BK));   // K steps come in pairs
  const int work = SPLIT ? tiles * splits : tiles;

  // Copies of codes: copy j of a half writes LDS rows [RPC x, RPC x + RPC), x = W j + wave; lane l
  // writes slot l % CPR of row l / CPR.  Half row r lies in wave block r / R of that half.
  const int lrow = lane / CPR;
  const int chunk = ((lane % CPR) ^ swz<BK>(wave * RPC + lrow)) * 16;
  static_assert((W * RPC) % 16 == 0, "the swizzle must not depend on j");
  const int lda32 = (int)p.lda, ldb32 = (int)p.ldb;
  int arow[2][JA], brow[2][JB[0]];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    constexpr int RA = 32 * QA;
#pragma unroll
    for (int j = 0; j < JA; ++j) {
      const int r = (W * j + wave) * RPC;
      arow[h][j] = (r / RA) * (2 * RA) + h * RA + r % RA;
    }
    const int RB = 32 * QB[h];
#pragma unroll
    for (int j = 0; j < JB[0]; ++j) {
      const int r = (W * j + wave) * RPC;
      brow[h][j] = ((r / RB) * (32 * QN) + h * 32 * QB0 + r % RB) * ldb32;
    }
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_i8*)lds + wave * 1024;
  const uint32_t voffB = (uint32_t)(lrow * ldb32 + chunk);
  uint32_t voffA[2][JA], voffS[JS];
  const uint8_t *pA, *pB;      // the K position being requested, in the tile being requested
  const uint8_t *psA, *psB;    // the batch of scales being requested
  int sreq = 0;                // its buffer (bytes from SC0)
  // the tile, the first K step and the number of steps of a piece of work
  auto work_at = [&](int piece, int64_t& mt, int64_t& nt, int& k0, int& kt) {
    const int tile = SPLIT ? piece % tiles : piece, part = SPLIT ? piece / tiles : 0;
    if constexpr (SPLIT) {
      const int most = pairs / splits, more = pairs % splits;
      k0 = 2 * (part * most + min(part, more));
      kt = 2 * (most + (part < more));
    } else {
      k0 = 0;
      kt = 2 * pairs;
    }
    int pid_m, pid_n;
    staged_tile(tiles % 8 == 0 ? tile : xcd_order(tile, tiles), tiles, num_pid_m, num_pid_n, group_m,
                pid_m, pid_n);
    mt = (int64_t)pid_m * BM;
    // the last column tile ends at N: columns it shares with the one before get the same values twice
    nt = min(pid_n * BN, N - BN);
  };
  // copy j of the batch: rows [64 x, 64 x + 64) of the tile's A rows and then B rows
  auto scale_copy = [&](int j) { return min(W * j + wave, SC - 1); };
  auto request_from = [&](int64_t mt, int64_t nt, int k0) {
    pA = p.a + mt * p.lda + (int64_t)k0 * BK;
    pB = p.b + nt * p.ldb + (int64_t)k0 * BK;
    psA = p.sa + mt * p.ldsa + k0 * 8;
    psB = p.sb + nt * p.ldsb + k0 * 8;
    const int last = M - 1 - (int)mt;   // token rows past M copy the last row, never stored
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < JA; ++j)
        voffA[h][j] = (uint32_t)(min(arow[h][j] + lrow, last) * lda32 + chunk);
#pragma unroll
    for (int j = 0; j < JS; ++j) {
      const int x = scale_copy(j);
      voffS[j] = (uint32_t)(x < BM / 64 ? min(64 * x + lane, last) * (int)p.ldsa
                                        : (64 * (x - BM / 64) + lane) * (int)p.ldsb);
    }
  };
  // copy j of A's / B's half h of the step at pA / pB, into buffer buf
  auto copyA = [&](int h, int buf, int j) {
    copy_1k(pA, voffA[h][j], lds0 + (2 * buf + h) * HA + j * 1024 * W);
  };
  auto copyB = [&](int h, int buf, int j) {
    copy_1k(pB + brow[h][j], voffB, lds0 + B0 + buf * SB + h * HB[0] + j * 1024 * W);
  };
  auto copyS = [&]() {
#pragma unroll
    for (int j = 0; j < JS; ++j) {
      const int x = scale_copy(j);
      copy_1k(x < BM / 64 ? psA : psB, voffS[j], lds0 - wave * 1024 + SC0 + sreq + x * 1024);
    }
    psA += 16;
    psB += 16;
    sreq ^= SCB;
  };

  // Fragment reads: lane l reads row l % 32 of a 32-row block, chunk 4 (l / 32) + kk.
  const int frow = lane & 31, fhalf = lane >> 5;
  int ofs[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) ofs[kk] = frow * BK + (((4 * fhalf + kk) ^ swz<BK>(frow)) * 16);
  const int8_t* la = lds + wm * 32 * QA * BK;
  const int8_t* lb[2] = {lds + B0 + wn * 32 * QB0 * BK, lds + B0 + HB[0] + wn * 32 * QB1 * BK};
  // scales: a row's 16 bytes are two steps of two words, one a half of the lanes
  const int8_t* lsa = lds + SC0 + (wm * 64 * QA + frow) * 16 + 4 * fhalf;
  const int8_t* lsb = lds + SC0 + (BM + wn * 32 * QN + frow) * 16 + 4 * fhalf;
  int sread = 0;               // the buffer of the step being multiplied
  v4i fa[2][QA][KK], fb[2][QB0][KK];
  int sca[2][QA], scb[2][QB0];
  // fragments of half h of the step in buffer buf (0: even), its scales in the current buffer or,
  // with `next`, in the other one
  auto readA = [&](int h, int buf, int kk, bool next) {
#pragma unroll
    for (int i = 0; i < QA; ++i) {
      fa[h][i][kk] = *(const v4i*)(la + ofs[kk] + (2 * buf + h) * HA + i * 32 * BK);
      if (kk == 0)
        sca[h][i] = *(const int*)(lsa + (next ? sread ^ SCB : sread) + 8 * buf + (h * QA + i) * 512);
    }
  };
  auto readB = [&](int h, int buf, int kk, bool next) {
#pragma unroll
    for (int i = 0; i < QB0; ++i)
      if (i < QB[h]) {
        fb[h][i][kk] = *(const v4i*)(lb[h] + ofs[kk] + buf * SB + i * 32 * BK);
        if (kk == 0)
          scb[h][i] =
              *(const int*)(lsb + (next ? sread ^ SCB : sread) + 8 * buf + (h * QB0 + i) * 512);
      }
  };

  v16f acc[2][2][QA][QB0];
  // A phase's work: per MFMA substep its MFMAs with the next phase's reads between them, and one in
  // KK of its copies.  zero: a tile's first step, which starts the sums from 0.
  auto body = [&](auto hac, auto hbc, auto zero, auto read, int reads, auto copy, auto copies) {
    constexpr int ha = decltype(hac)::value, hb = decltype(hbc)::value;
    constexpr int NC = decltype(copies)::value;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
      for (int i = 0; i < QA; ++i)
#pragma unroll
        for (int j = 0; j < QB[hb]; ++j)
          acc[ha][hb][i][j] = mx_mfma(fb[hb][j][kk], fa[ha][i][kk],
                                      decltype(zero)::value && kk == 0 ? v16f{} : acc[ha][hb][i][j],
                                      scb[hb][j], sca[ha][i], kk);
      if (kk < 2) {   // in the first two substeps, so that the last two's MFMAs cover their way back
        read(2 * kk);
        read(2 * kk + 1);
      }
#pragma unroll
      for (int j = kk * NC / KK; j < (kk + 1) * NC / KK; ++j) copy(j);
#pragma unroll
      for (int i = 0; i < QA * QB[hb]; ++i) {
        // an MFMA, then its share of the reads
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (kk < 2 && i < 2 * reads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (kk < 2 && QA * QB[hb] + i < 2 * reads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // One K step of parity `par`.  TAIL: a tile's last (it reads nothing ahead).  HEAD: 4 for a
  // tile's first step and 1 for its second, the phases that `landed` spares the wait for copies
  // (a workgroup's later tiles find them landed).
  auto step = [&](auto par, auto tail, auto headc, bool landed) {
    constexpr int f = decltype(par)::value, s = 1 - f;
    constexpr bool TAIL = decltype(tail)::value;
    constexpr int HEAD = decltype(headc)::value;
    constexpr std::bool_constant<HEAD == 4> zero{};
    typedef std::integral_constant<int, 0> H0;
    typedef std::integral_constant<int, 1> H1;
    typedef std::integral_constant<int, f> HF;
    typedef std::integral_constant<int, s> HS;
    // the copies that may be in flight at a phase's end: the newest five halves, and a batch of
    // scales requested among them (by this step, or before phase 0's by the step before)
    constexpr int NA = 3 * JA + JB[0] + JB[1], NB = 2 * JA + JB[0] + JB[1] + JB[f];
    auto phase_end = [&](auto phasec, auto nc) {
      constexpr int phase = decltype(phasec)::value;
      constexpr int N = decltype(nc)::value + (phase == 0 || f == 0 ? JS : 0);
      if constexpr (phase < HEAD) {
        wait_lgkmcnt0();
        if (!landed) wait_vmcnt<N>();
      } else {
        wait_vmcnt_lgkm0<N>();
      }
      lds_barrier();
    };
    // opaque to the compiler, so that it keeps them in scalar registers
    asm volatile("" : "+s"(pA), "+s"(pB));
    if constexpr (f == 0) copyS();
    constexpr bool next = f == 1;   // the step after this one has its scales in the other buffer
    body(H0{}, HF{}, zero, [&](int kk) { readB(s, f, kk, false); }, QB[s],
         [&](int j) { copyA(0, f, j); }, std::integral_constant<int, JA>{});
    phase_end(std::integral_constant<int, 0>{}, std::integral_constant<int, NA>{});

    body(H0{}, HS{}, zero, [&](int kk) { readA(1, f, kk, false); }, QA,
         [&](int j) { copyB(f, f, j); }, std::integral_constant<int, JB[f]>{});
    phase_end(std::integral_constant<int, 1>{}, std::integral_constant<int, NB>{});

    body(H1{}, HS{}, zero, [&](int kk) { if constexpr (!TAIL) readA(0, 1 - f, kk, next); },
         TAIL ? 0 : QA, [&](int j) { copyB(s, f, j); }, std::integral_constant<int, JB[s]>{});
    if constexpr (!TAIL) phase_end(std::integral_constant<int, 2>{}, std::integral_constant<int, NB>{});

    body(H1{}, HF{}, zero, [&](int kk) { if constexpr (!TAIL) readB(s, 1 - f, kk, next); },
         TAIL ? 0 : QB[s], [&](int j) { copyA(1, f, j); }, std::integral_constant<int, JA>{});
    if constexpr (!TAIL) phase_end(std::integral_constant<int, 3>{}, std::integral_constant<int, NA>{});
    pA += BK;
    pB += BK;
    if constexpr (f == 1) sread ^= SCB;
  };
  typedef std::integral_constant<int, 0> P0;
  typedef std::integral_constant<int, 1> P1;
  auto request_step = [&](auto par) {   // a whole step, in the order the phases request it
    constexpr int f = decltype(par)::value, s = 1 - f;
    for (int j = 0; j < JA; ++j) copyA(0, f, j);
    for (int j = 0; j < JB[f]; ++j) copyB(f, f, j);
    for (int j = 0; j < JB[s]; ++j) copyB(s, f, j);
    for (int j = 0; j < JA; ++j) copyA(1, f, j);
    pA += BK;
    pB += BK;
  };

  int piece = blockIdx.x, k0, KT;
  int64_t m0, n0;
  work_at(piece, m0, n0, k0, KT);
  request_from(m0, n0, k0);
  copyS();
  request_step(P0{});
  request_step(P1{});
  bool landed = false;
  for (;;) {
    // A0(0) and B0(0) into registers, then the steps in pairs, the first and the last apart
    if (!landed) wait_vmcnt<3 * JA + JB[0] + 2 * JB[1]>();
    lds_barrier();
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      readA(0, 0, kk, false);
      readB(0, 0, kk, false);
    }
    wait_lgkmcnt0();
    if (!landed) wait_vmcnt<3 * JA + JB[0] + JB[1]>();
    lds_barrier();

    const int next = piece + gridDim.x;   // past the last piece: its own start again, not used
    int64_t m1 = m0, n1 = n0;
    int k1 = k0, KT1 = KT;
    if (next < work) work_at(next, m1, n1, k1, KT1);
    step(P0{}, std::false_type{}, std::integral_constant<int, 4>{}, landed);
    step(P1{}, std::false_type{}, std::integral_constant<int, 1>{}, landed);
    for (int t = 2; t + 2 < KT; t += 2) {
      step(P0{}, std::false_type{}, P0{}, false);
      step(P1{}, std::false_type{}, P0{}, false);
    }
    request_from(m1, n1, k1);
    step(P0{}, std::false_type{}, P0{}, false);
    step(P1{}, std::true_type{}, P0{}, false);
    // the sums stay in AGPRs up to here: with the epilogue's use of them in sight, the compiler
    // moves the last steps' into VGPRs and spills 120 others (256 x 256)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int hb = 0; hb < 2; ++hb)
#pragma unroll
        for (int i = 0; i < QA; ++i)
#pragma unroll
          for (int j = 0; j < QB[hb]; ++j) asm volatile("" : "+a"(acc[h][hb][i][j]));

    // ---- epilogue: the bias in fp32, one cast.  Each wave takes 32 tokens x 64 columns (16-bit
    // outputs; 32 columns of 4-byte ones) at a time through its 4 KiB: rows of 128 bytes, chunk c
    // at slot c ^ (row & 7), written out in whole 128-byte lines, 8 rows a store.  The lane index
    // is taken anew, opaque, so that what the epilogue derives from it is not kept in registers
    // over the main loop.
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int erow = ln & 31, ehalf = ln >> 5, srow = ln >> 3, sch = ln & 7;
    const int64_t nw = n0 + wn * 32 * QN, mw = m0 + wm * 64 * QA;
    int8_t* stg = lds + STG + wave * 4096;
    float* plane = SPLIT ? (float*)p.out + (int64_t)(piece / tiles) * M * p.ldc : (float*)p.out;
#pragma unroll
    for (int g = 0; g < (QN + 1) / 2; ++g) {   // fragments 2g and 2g+1 of the wave's columns
      const int nf = QN % 2 == 1 && g == QN / 2 ? 1 : 2;   // (an odd last fragment stands alone)
      float bias[2][4][4];
      if constexpr (BIAS) {
#pragma unroll
        for (int c = 0; c < nf; ++c)
#pragma unroll
          for (int q = 0; q < 4; ++q) bias4(p, nw + 64 * g + 32 * c + 8 * q + 4 * ehalf, bias[c][q]);
      }
      if (g == 0) {
        // every copy in flight (the next tile's first two steps) has landed past here, so the
        // next tile's first waits need not count past this tile's stores
        wait_vmcnt<0>();
        asm volatile("" ::: "memory");
      }
      auto value = [&](int h, int i, int c, int q, int r) {
        const int x = 2 * g + c, hb = x >= QB0;
        const float v = acc[h][hb][i][x - hb * QB0][4 * q + r];
        return BIAS ? v + bias[c][q][r] : v;
      };
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < QA; ++i) {
          const int64_t mb = mw + (h * QA + i) * 32;
          if constexpr (OD == I8L_F32) {
#pragma unroll
            for (int c = 0; c < nf; ++c) {
              const int x = 2 * g + c;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                v4f v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = value(h, i, c, q, r);
                *(v4f*)(stg + erow * 128 + (((2 * q + ehalf) ^ (erow & 7)) * 16)) = v;
              }
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const int row = 8 * y + srow;
                const v4i v = *(const v4i*)(stg + row * 128 + ((sch ^ srow) * 16));
                v4i* at = (v4i*)(plane + (mb + row) * p.ldc + nw + 32 * x + 4 * sch);
                if (mb + row < M) {
                  if constexpr (SPLIT) *at = v;   // read again at once
                  else __builtin_nontemporal_store(v, at);
                }
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < nf; ++c)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = value(h, i, c, q, r);
                *(uint2*)(stg + erow * 128 + (((4 * c + q) ^ (erow & 7)) * 16) + 8 * ehalf) =
                    make_uint2(f32x2_to_act2<OD>(v[0], v[1]), f32x2_to_act2<OD>(v[2], v[3]));
              }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int row = 8 * y + srow;
              const v4i v = *(const v4i*)(stg + row * 128 + ((sch ^ srow) * 16));
              if (mb + row < M && (nf == 2 || sch < 4))
                __builtin_nontemporal_store(
                    v, (v4i*)((uint16_t*)p.out + (mb + row) * p.ldc + nw + 64 * g + 8 * sch));
            }
          }
        }
      asm volatile("" ::: "memory");   // the next 64 columns' operands load after these
    }
    if (next >= work) break;
    piece = next;
    m0 = m1;
    n0 = n1;
    k0 = k1;
    KT = KT1;
    landed = true;
  }
}

// The sum of the parts' planes in order, the bias and one rounding; a thread four columns.
template <int OD>
__global__ void __launch_bounds__(256) mxfp4_sum_parts(MxMM p, const float* __restrict__ parts,
                                                       int splits) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, plane = p.M * p.N;
  if (i >= plane) return;
  v4f v = *(const v4f*)(parts + i);
  for (int z = 1; z < splits; ++z) v += *(const v4f*)(parts + z * plane + i);
  const int64_t m = i / p.N, n = i % p.N;
  if (p.bias) {
    float b[4];
    bias4(p, n, b);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += b[r];
  }
  if constexpr (OD == I8L_F32) {
    *(v4f*)((float*)p.out + m * p.ldc + n) = v;
  } else {
    *(uint2*)((uint16_t*)p.out + m * p.ldc + n) =
        make_uint2(f32x2_to_act2<OD>(v[0], v[1]), f32x2_to_act2<OD>(v[2], v[3]));
  }
}

// ------------------------------------------------------------------ host side
// The tiles, and what a piece of work on one was measured to take (us): a K step with the card
// nearly idle and with a piece on every CU (the clock falls as the card fills), and the rest.
struct PhasedTile {
  int bm, bn;
  float step_idle, step_full, rest;
};
constexpr PhasedTile kTiles[] = {{256, 256, 1.04f, 1.72f, 4.5f}, {256, 192, 0.94f, 1.35f, 4.0f},
                                 {256, 128, 0.75f, 1.05f, 2.8f}, {128, 256, 0.87f, 1.05f, 2.8f},
                                 {128, 192, 0.78f, 0.88f, 2.5f}, {128, 128, 0.66f, 0.72f, 1.2f}};

template <int QA, int QB0, int QB1, int OD, bool BIAS, bool SPLIT>
hipError_t launch_phased_k(const MxMM& p, int splits, hipStream_t st) {
  auto kern = mxfp4_phased<QA, QB0, QB1, OD, BIAS, SPLIT>;
  constexpr int BM = 128 * QA, BN = 64 * (QB0 + QB1);
  constexpr size_t shm = 2 * (size_t)(BM + BN) * (128 + 16) + 4 * 4096;
  static_assert(shm <= kMaxLds, "two buffers, two batches of scales and the staging fit the LDS");
  static std::atomic<uint64_t> lds_done{0};
  lds_opt_in((const void*)kern, shm, lds_done);
  const int tiles = (int)((p.M + BM - 1) / BM * ((p.N + BN - 1) / BN));
  const int grid = std::min(tiles * splits, cu_count() * (int)(kMaxLds / shm));
  // 8 rows of tiles walked together (4096 x 28672: 2 rows 226 us, 4 222, 8 221, 16 223)
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), shm, st, p, 8, tiles, splits);
  return hipGetLastError();
}

template <int QA, int QB0, int QB1>
hipError_t launch_phased_t(const MxMM& p, int splits, float* parts, hipStream_t st) {
  if (splits > 1) {
    MxMM q = p;
    q.out = parts, q.ldc = p.N, q.out_dtype = I8L_F32, q.bias = nullptr;
    const hipError_t e = launch_phased_k<QA, QB0, QB1, I8L_F32, false, true>(q, splits, st);
    if (e) return e;
    const dim3 grid((unsigned)((p.M * p.N + 1023) / 1024));
    auto sum = p.out_dtype == I8L_BF16  ? mxfp4_sum_parts<I8L_BF16>
               : p.out_dtype == I8L_F16 ? mxfp4_sum_parts<I8L_F16>
                                        : mxfp4_sum_parts<I8L_F32>;
    hipLaunchKernelGGL(sum, grid, dim3(256), 0, st, p, parts, splits);
    return hipGetLastError();
  }
  auto go = [&](auto odc) {
    constexpr int OD = decltype(odc)::value;
    return p.bias ? launch_phased_k<QA, QB0, QB1, OD, true, false>(p, 1, st)
                  : launch_phased_k<QA, QB0, QB1, OD, false, false>(p, 1, st);
  };
  switch (p.out_dtype) {
    case I8L_BF16: return go(std::integral_constant<int, I8L_BF16>{});
    case I8L_F16: return go(std::integral_constant<int, I8L_F16>{});
  }
  return go(std::integral_constant<int, I8L_F32>{});
}

}  // namespace

bool mx_phased_ok(const MxMM& p) {
  const int es = elt_size(p.out_dtype);
  return aligned16(p.a) && aligned16(p.b) && aligned16(p.sa) && aligned16(p.sb) && aligned16(p.out) &&
         (!p.bias || aligned16(p.bias)) && p.lda % 16 == 0 && p.ldb % 16 == 0 && p.ldsa % 16 == 0 &&
         p.ldsb % 16 == 0 && p.ldc * es % 16 == 0 && p.K % 512 == 0 && p.K >= 1024 && p.N % 8 == 0 &&
         p.N >= 128 && p.lda <= 1 << 22 && p.ldb <= 1 << 22 && p.ldsa <= 1 << 22 &&
         p.ldsb <= 1 << 22 && p.M < (int64_t)1 << 30 && p.N < (int64_t)1 << 30 &&
         (p.M + 127) / 128 * ((p.N + 127) / 128) < (int64_t)1 << 26;
}

hipError_t launch_mx_phased_tile(int t, int splits, float* parts, const MxMM& p, hipStream_t st) {
  switch (t) {
    case 0: return launch_phased_t<2, 2, 2>(p, splits, parts, st);
    case 1: return launch_phased_t<2, 2, 1>(p, splits, parts, st);
    case 2: return launch_phased_t<2, 1, 1>(p, splits, parts, st);
    case 3: return launch_phased_t<1, 2, 2>(p, splits, parts, st);
    case 4: return launch_phased_t<1, 2, 1>(p, splits, parts, st);
  }
  return launch_phased_t<1, 1, 1>(p, splits, parts, st);
}

// The tile and the parts of K with the least modelled time: rounds of a piece on every CU, each the
// piece's steps and rest, and for parts the sum's launch and traffic (S planes written and read at
// 4.4 TB/s).  Measured against it (cold weights, us; unsplit / split): 14336 -> 4096 at 128 tokens
// 30 / 17.8 in 7 parts, at 256 33 / 22.7 in 4, at 512 41.8 / 31.7 in 2; 2048 -> 4096 at 512 6.9 / 18.4.
MxPhasedPlan mx_phased_plan(int64_t M, int64_t N, int64_t K, int64_t workspace) {
  MxPhasedPlan best{-1, 1, 0, 0};
  double least = 0;
  const int64_t pairs = K / 512;
  const int cus = 256;
  for (int t = 0; t < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++t) {
    const PhasedTile& tile = kTiles[t];
    if (N < tile.bn) continue;
    const int64_t tiles = (M + tile.bm - 1) / tile.bm * ((N + tile.bn - 1) / tile.bn);
    for (int64_t s = 1; s <= kMaxParts && 2 * s <= pairs; ++s) {
      if (s > 1 && (s * M * N * 4 > workspace || tiles * s > cus)) break;
      const double steps = 2.0 * ((pairs + s - 1) / s);
      const int64_t work = tiles * s, rest = work % cus;
      const double load = (double)rest / cus;
      double us = (double)(work / cus) * (steps * tile.step_full + tile.rest);
      if (rest)
        us += steps * (tile.step_idle + (tile.step_full - tile.step_idle) * load) + tile.rest;
      if (s > 1) us += 2.5 + 8.0 * s * M * N / 4.4e6;
      if (best.tile < 0 || us < least) best = {t, (int)s, tile.bm, tile.bn}, least = us;
    }
  }
  return best;
}

hipError_t launch_mx_phased(const MxMM& p, void* workspace, int64_t bytes, hipStream_t st) {
  const MxPhasedPlan plan =
      mx_phased_plan(p.M, p.N, p.K, workspace && aligned16(workspace) ? bytes : 0);
  return launch_mx_phased_tile(plan.tile, plan.splits, (float*)workspace, p, st);
}

}  // namespace i8l
