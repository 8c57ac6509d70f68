// Macro tiles of the grouped W8A8 product, for experts with many rows: persistent workgroups whose K
// steps are cut into four phases, one per quadrant of a wave's tile (v_mfma_i32_32x32x32_i8).
#include "i8l_gemm_tile.h"
#include "i8l_grouped.h"

namespace i8l {

namespace {

// ------------------------------------------------------------------ schedule
// A workgroup of 4 waves (WM x WN, one a SIMD) computes BM x BN tiles in 128-byte K steps.  A wave's
// tile is 2 x 2 quadrants of 32 x 32 fragments: its rows are an A half 0 and 1 of QA fragments each,
// its columns a B half 0 and 1 of QB each, and the LDS holds each operand's step as those two halves
// in two buffers.  With SILU the B half 0 is gate columns and half 1 the up columns of the same
// indices, so a lane ends with both factors of its outputs.
//
// Step t is four phases, with f = t % 2 and s = 1 - f (the order of the B halves alternates):
//   phase 0: MFMAs of (A0, Bf);   reads Bs(t);     requests A0(t+2)
//   phase 1: MFMAs of (A0, Bs);   reads A1(t);     requests Bf(t+2)
//   phase 2: MFMAs of (A1, Bs);   reads A0(t+1);   requests Bs(t+2)
//   phase 3: MFMAs of (A1, Bf);   reads Bs(t+1), which is t+1's first;  requests A1(t+2)
// so every fragment is read from LDS once a step and a phase before its use, and the copies of a step
// go out a quarter a phase, each into the half whose reads ended a phase before, six phases before it
// is read.  Each phase ends with lgkmcnt(0) (this wave's reads are done: that half may be refilled),
// vmcnt (all but the newest five halves have landed: the next phase's reads) and one workgroup
// barrier, which makes both true of every wave.
//
// A half is BM / 2 rows in a row, so a tile of no more rows than that (an expert's last) leaves out the
// MFMAs of phases 2 and 3.
//
// The workgroups walk the tiles of all experts; the copies of a tile's last two steps are the next
// tile's first two, so they fly during the epilogue, which every wave does alone through its own 4 KiB
// of LDS.  What the epilogue reads stands in LDS before it begins (the tile's scales and bias, and the
// experts' first blocks and rows, by which tiles are found), since a wait for a load would be one for
// the copies requested before it; it is fetched an epilogue ahead, the rows' indices two, behind the
// copies and awaited with them when half of the stores are out.
//
// Rows past the expert's last, whole steps past K and its tail within a step are read outside the
// buffers, as zeros, at the price of one instruction a copy (zeros toggle nothing: they cost little of
// the power that bounds the multiplications).
//
// What bounds it: from about 1000 rows an expert the power, as in the dense tile (8 experts of 1024,
// 4096 -> 28672, tiles of 256 rows: 781 us, 2.46 POP/s, clock 1.55 GHz at 67% MFMA busy).  With fewer rows
// and shorter K, that a CU holds one workgroup and a SIMD one wave, so that nothing multiplies during an
// epilogue (256 x 256: 6.5 us of 34 at a K of 2048, its 128 KB stored at 5.1 TB/s by all CUs at a time; with
// SILU 7.2, exp and reciprocal): 128 experts of 512 rows, 2048 -> 1536, 206 us, 2.0 POP/s.  4096 tokens'
// 32768 rows, 1 to 1400 an expert, with SILU: 148 us, 1.4 POP/s, MFMA busy 40%; a fifth of the rows it
// multiplies are an expert's last tile's padding, and an even deal of the tiles to workgroups won 1% of it.
// Below about 100 rows the weight stream (32 rows of each of 128: 72 us for 403 MB, 5.6 TB/s).
constexpr int kStep = 128;

constexpr int kTiles = 32;   // found half of them at a time, a tile a lane

struct PhasedShared {
  int32_t first[kMaxExperts + 1];            // an expert's first block; [E]: their number
  int32_t lo[kMaxExperts], hi[kMaxExperts];  // its rows
  int32_t source[3][256];                    // a tile's rows of A; -1: past the expert's last
  GroupTile tile[kTiles];                    // the workgroup's tiles, its nth in slot n % kTiles
  alignas(16) float sa[2][256], sb[2][256], bias[2][256];   // a tile's rows' and columns'
};

constexpr int kStoreCpol = 2;   // non-temporal: the next kernel's reads, if any, are far behind

// The lane's number, counted where it is asked for: a value derived from it there is neither kept in
// registers over the main loop nor, worse, out of them (a reload waits for the copies in flight).
__device__ __forceinline__ int fresh_lane() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(l));
  return l;
}

// p[i] by a scalar base and a 32-bit byte offset.
template <typename T>
__device__ __forceinline__ T at32(const T* p, int i) {
  return *(const T*)((const char*)p + (uint32_t)i * (uint32_t)sizeof(T));
}

constexpr int kBadRow = -2;   // a source row outside [0, M): zeros, and NaN in the end

// STREAM: the weights are not kept in the caches, as most experts' are read by one row block only.
template <int WM, int QA, int QB, int OD, bool BIAS, bool SILU, bool STREAM>
__global__ void __launch_bounds__(256) grouped_phased(Grouped p, uint32_t abytes, uint32_t bbytes, int steps) {
  constexpr int W = 4, WN = W / WM;
  constexpr int QN = 2 * QB;                         // column fragments of a wave
  constexpr int BM = WM * 64 * QA, BN = WN * 32 * QN, BK = kStep;
  constexpr int BNO = SILU ? BN / 2 : BN;            // output columns
  static_assert(BN == 256 && BM <= 256, "a thread a row and a column");
  constexpr int CPR = BK / 16, RPC = 64 / CPR;       // chunks of a row, rows of a copy
  constexpr int KK = BK / 32;                        // MFMA substeps of a step
  constexpr int HA = BM / 2 * BK, HB = BN / 2 * BK;  // bytes of a half
  constexpr int JA = HA / 1024 / W, JB = HB / 1024 / W;   // copies a wave
  constexpr int B0 = 4 * HA, SB = 2 * HB;            // LDS: A [buffer][half], then B, then staging
  constexpr int STG = B0 + 2 * SB;
  static_assert(JA >= 1 && JB >= 1, "whole copies");
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  PhasedShared& sh = *(PhasedShared*)(lds + STG + W * 4096);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int width = SILU ? p.N / 2 : p.N;            // output columns of the problem
  const int cols = (width + BNO - 1) / BNO;
  const int KT = steps;

  // ---- the experts' blocks
  if (wave == 0) {
    int lowest = 0, before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
      const int e = min(e0 + lane, p.E - 1);
      const bool in = e0 + lane < p.E;
      const ExpertRows x = expert_rows(p, BM, in, p.offsets[e], p.offsets[e + 1], lowest, before);
      if (in) {
        sh.lo[e] = x.lo;
        sh.hi[e] = x.hi;
        sh.first[e] = x.upto - x.blocks;
      }
    }
    if (lane == 0) sh.first[p.E] = before;
  }
  __syncthreads();
  const int total_blocks = __builtin_amdgcn_readfirstlane(sh.first[p.E]);
  const int64_t total64 = (int64_t)total_blocks * cols;
  const int tiles = __builtin_amdgcn_readfirstlane((int)min(total64, (int64_t)INT32_MAX));
  if ((int)blockIdx.x >= tiles) return;
  const int stride = gridDim.x;

  // Tile t of all: consecutive positions go to one XCD, and within an expert up to 8 row blocks
  // are walked together, so that what runs at a time shares weight and activation rows in L2.  Each
  // round of an XCD's workgroups is turned by one against the last, so that none of them meets only
  // full tiles and none only last ones.
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };   // (it is: said to the compiler)
  const int group = stride / 8;
  auto tile_at = [&](int t) {   // t: a lane's own
    const int round = group ? t / 8 / group : 0;
    if (group && stride % 8 == 0 && (round + 1) * group * 8 <= tiles)
      t = (round * group + (t / 8 + round) % group) * 8 + t % 8;
    const int pos = xcd_order(t, tiles);
    const int q = pos / cols;
    GroupTile o;
    o.e = 0;                    // the last expert whose first block is not behind q
#pragma unroll
    for (int step = kMaxExperts / 2; step; step /= 2)
      if (o.e + step < p.E && sh.first[o.e + step] <= q) o.e += step;
    const int f = sh.first[o.e], nb = sh.first[o.e + 1] - f;
    const int local = pos - f * cols;
    constexpr int GM = 8;
    const int first = local / (GM * cols) * GM, gsize = min(nb - first, GM);
    const int in = local - first * cols;
    o.col = in / gsize;
    o.row0 = sh.lo[o.e] + (first + in % gsize) * BM;
    o.end = min(o.row0 + BM, sh.hi[o.e]);
    return o;
  };
  // The workgroup's tiles n .. n + count - 1 into the table, by one wave; past the last: the last again.
  auto find_tiles = [&](int n, int count, int l) {
    if (l < count) {
      const int last = (tiles - 1 - (int)blockIdx.x) / stride;
      sh.tile[(n + l) % kTiles] = tile_at(blockIdx.x + min(n + l, last) * stride);
    }
  };
  // a tile's source rows: row x of it
  auto source_of = [&](const GroupTile& g, int x) {
    if (x >= BM) return -1;
    const int i = g.row0 + x;
    if (i >= g.end) return -1;
    const int r = p.rows ? at32(p.rows, i) : i;
    return r >= 0 && r < p.M ? r : kBadRow;
  };

  // Copies: copy j of a half writes LDS rows [RPC x, RPC x + RPC), x = W j + wave; lane l writes
  // slot l % CPR of row l / CPR.  B's half row r lies in wave block r / R of that half (R rows each).
  static_assert((W * RPC) % 16 == 0, "the swizzle must not depend on j");
  const int lda32 = (int)p.lda, ldb32 = (int)p.ldb;
  int brow[2][JB];         // the weight's byte offsets in the tile being requested
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_i8*)lds + wave * 1024;
  int lrow, chunk;
  uint32_t voffB;
  const v4u bufA = buffer_of(p.a, abytes);
  v4u bufB = bufA;
  uint32_t voffA[2][JA];
  int kreq, kat;           // the K position being requested; 0 for it past K, where nothing is read
  uint32_t past = 0;       // kOutside in the lanes whose chunk of that step lies past K
  // (found again at the start of the tile, rather than kept over the epilogue)
  auto request_from = [&](const GroupTile& g, int buf, int k) {
    kreq = k;
    bufB = buffer_of(p.b + g.e * p.eb, bbytes);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < JA; ++j) {
        const int r = sh.source[buf][h * (BM / 2) + (W * j + wave) * RPC + lrow];
        voffA[h][j] = r >= 0 ? (uint32_t)(r * lda32 + chunk) : kOutside;
      }
      constexpr int RB = 32 * QB;
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        // eight columns, all within the problem or all past it (then the last eight again, not stored)
        const int r = (W * j + wave) * RPC, x = r / RB, y = r % RB;
        const int n = SILU ? h * width + min(g.col * BNO + x * RB + y, width - 8)
                           : min(g.col * BN + x * (2 * RB) + h * RB + y, width - 8);
        brow[h][j] = uniform(n * ldb32);
      }
    }
  };
  auto begin_step = [&] {
    past = kreq + chunk < p.K ? 0u : kOutside;
    kat = kreq < p.K ? kreq : 0;   // (so that the scalar offset stays within the buffer)
  };
  // copy j of A's / B's half h of the step being requested, into buffer buf
  auto copyA = [&](int h, int buf, int j) {
    copy_1k(bufA, voffA[h][j] | past, kat, lds0 + (2 * buf + h) * HA + j * 1024 * W);
  };
  auto copyB = [&](int h, int buf, int j) {
    const uint32_t dst = lds0 + B0 + buf * SB + h * HB + j * 1024 * W;
    if constexpr (STREAM) copy_1k_stream(bufB, voffB | past, kat + brow[h][j], dst);
    else copy_1k(bufB, voffB | past, kat + brow[h][j], dst);
  };

  // Fragment reads: lane l reads row l%32 of a 32-row block, chunk 2*kk + l/32.
  int ofs[KK];
  // what the main loop derives from the lane, anew for each tile
  auto lay_out = [&] {
    const int l = fresh_lane();
    lrow = l / CPR;
    chunk = ((l % CPR) ^ swz<BK>(wave * RPC + lrow)) * 16;
    voffB = (uint32_t)(lrow * ldb32 + chunk);
    const int frow = l & 31, fhalf = l >> 5;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) ofs[kk] = frow * BK + (((2 * kk + fhalf) ^ swz<BK>(frow)) * 16);
  };
  const int8_t* la = lds + wm * 32 * QA * BK;
  const int8_t* lb = lds + B0 + wn * 32 * QB * BK;
  v4i fa[2][QA][KK], fb[2][QB][KK];
  auto readA = [&](int h, int buf, int kk) {
#pragma unroll
    for (int i = 0; i < QA; ++i)
      fa[h][i][kk] = *(const v4i*)(la + ofs[kk] + (2 * buf + h) * HA + i * 32 * BK);
  };
  auto readB = [&](int h, int buf, int kk) {
#pragma unroll
    for (int i = 0; i < QB; ++i)
      fb[h][i][kk] = *(const v4i*)(lb + ofs[kk] + buf * SB + h * HB + i * 32 * BK);
  };

  // A phase's work: per MFMA substep its MFMAs with the next phase's reads of that substep between
  // them, and one in KK of its copies.  zero: a tile's first step, whose first substep starts from 0.
  typedef v16i Sums[2][2][QA][QB];
  auto body = [&](Sums& acc, auto hac, auto hbc, auto fullc, auto zero, auto read, int reads, auto copy, auto copies) {
    constexpr int ha = decltype(hac)::value, hb = decltype(hbc)::value;
    constexpr int NC = decltype(copies)::value;
    if constexpr (ha == 1 && !decltype(fullc)::value) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) read(kk);
#pragma unroll
      for (int j = 0; j < NC; ++j) copy(j);
      return;
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
      for (int i = 0; i < QA; ++i)
#pragma unroll
        for (int j = 0; j < QB; ++j)
          acc[ha][hb][i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
              fb[hb][j][kk], fa[ha][i][kk],
              decltype(zero)::value && kk == 0 ? v16i{} : acc[ha][hb][i][j], 0, 0, 0);
      read(kk);
#pragma unroll
      for (int j = kk * NC / KK; j < (kk + 1) * NC / KK; ++j) copy(j);
#pragma unroll
      for (int i = 0; i < QA * QB; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                 // one MFMA
        if (i < reads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // one LDS read
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // One K step of parity `par`.  TAIL: a tile's last (it reads nothing ahead).  HEAD: 4 for a
  // tile's first step and 1 for its second, the phases that `landed` spares the wait for copies
  // (a workgroup's later tiles find them landed).  fullc: the tile has rows in A's half 1.
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  typedef std::integral_constant<int, JA> NJA;
  typedef std::integral_constant<int, JB> NJB;
  auto step = [&](Sums& acc, auto par, auto tail, auto headc, auto fullc, bool landed) {
    constexpr int f = decltype(par)::value, s = 1 - f;
    constexpr bool TAIL = decltype(tail)::value;
    constexpr int HEAD = decltype(headc)::value;
    constexpr std::bool_constant<HEAD == 4> zero{};
    typedef std::integral_constant<int, f> HF;
    typedef std::integral_constant<int, s> HS;
    constexpr int NA = 3 * JA + 2 * JB, NB = 2 * JA + 3 * JB;
    auto phase_end = [&](auto phasec, auto nc) {
      constexpr int phase = decltype(phasec)::value, N = decltype(nc)::value;
      if constexpr (phase < HEAD) {
        wait_lgkmcnt0();
        if (!landed) wait_vmcnt<N>();
      } else {
        wait_vmcnt_lgkm0<N>();
      }
      lds_barrier();
    };
    begin_step();
    body(acc, I0{}, HF{}, fullc, zero, [&](int kk) { readB(s, f, kk); }, QB, [&](int j) { copyA(0, f, j); }, NJA{});
    phase_end(I0{}, std::integral_constant<int, NA>{});
    body(acc, I0{}, HS{}, fullc, zero, [&](int kk) { readA(1, f, kk); }, QA, [&](int j) { copyB(f, f, j); }, NJB{});
    phase_end(I1{}, std::integral_constant<int, NB>{});
    body(acc, I1{}, HS{}, fullc, zero, [&](int kk) { if constexpr (!TAIL) readA(0, 1 - f, kk); }, TAIL ? 0 : QA,
         [&](int j) { copyB(s, f, j); }, NJB{});
    if constexpr (!TAIL) phase_end(std::integral_constant<int, 2>{}, std::integral_constant<int, NB>{});
    body(acc, I1{}, HF{}, fullc, zero, [&](int kk) { if constexpr (!TAIL) readB(s, 1 - f, kk); }, TAIL ? 0 : QB,
         [&](int j) { copyA(1, f, j); }, NJA{});
    if constexpr (!TAIL) phase_end(std::integral_constant<int, 3>{}, std::integral_constant<int, NA>{});
    kreq += BK;
  };
  auto request_step = [&](auto par) {   // a whole step, in the order the phases request it
    constexpr int f = decltype(par)::value, s = 1 - f;
    begin_step();
    for (int j = 0; j < JA; ++j) copyA(0, f, j);
    for (int j = 0; j < JB; ++j) copyB(f, f, j);
    for (int j = 0; j < JB; ++j) copyB(s, f, j);
    for (int j = 0; j < JA; ++j) copyA(1, f, j);
    kreq += BK;
  };

  auto nth_tile = [&](int n) {
    const GroupTile& t = sh.tile[n % kTiles];
    return GroupTile{uniform(t.e), uniform(t.row0), uniform(t.end), uniform(t.col)};
  };
  // a tile's scales and bias: row x's, column x's
  struct Operands {
    float sa, sb;
    uint32_t bias;
  };
  auto operands_of = [&](const GroupTile& g, int source, int x) {
    Operands o;
    o.sa = at32(p.sa, p.sa_per_row ? max(source, 0) : 0);
    int n = g.col * BNO + x % BNO;
    n = min(n, width - 1) + (SILU && x >= BNO ? width : 0);
    const int64_t at = (int64_t)g.e * p.N;
    o.sb = at32(p.sb + at, n);
    o.bias = 0;
    if constexpr (BIAS)
      o.bias = p.bias_dtype == I8L_F32 ? at32((const uint32_t*)p.bias + at, n)
                                       : (uint32_t)at32((const uint16_t*)p.bias + at, n);
    return o;
  };
  auto keep = [&](int half, int source, const Operands& o, int x) {
    if (x < BM) sh.sa[half][x] = source == kBadRow ? __builtin_nanf("") : o.sa;
    sh.sb[half][x] = o.sb;
    if constexpr (BIAS)
      sh.bias[half][x] =
          p.bias_dtype == I8L_F32 ? __uint_as_float(o.bias) : act_to_f32(o.bias, p.bias_dtype);
  };
  if (wave == 0) find_tiles(0, kTiles, lane);
  __syncthreads();
  {
    const GroupTile g0 = nth_tile(0), g1 = nth_tile(1);
    const int s0 = source_of(g0, tid), s1 = source_of(g1, tid);
    keep(0, s0, operands_of(g0, s0, tid), tid);
    if (tid < BM) {
      sh.source[0][tid] = s0;
      sh.source[1][tid] = s1;
    }
    __syncthreads();
    lay_out();
    request_from(g0, 0, 0);
    request_step(I0{});
    request_step(I1{});
  }
  // The workgroup's nth tile, up to the start of the next.  fullc: it has rows in A's half 1.  Slots
  // n % 3 and n % 2 of the rows' and operands' tables are its own.
  auto run_tile = [&](auto fullc, const GroupTile& g0, int n) {
    const int rows = g0.end - g0.row0, half = n & 1;
    const int buf = n % 3, buf1 = (n + 1) % 3, buf2 = (n + 2) % 3;
    const bool landed = n > 0;
    lay_out();
    request_from(g0, buf, 2 * BK);
    // A0(0) and B0(0) into registers, then the steps in pairs, the first and the last apart
    if (!landed) wait_vmcnt<3 * JA + 3 * JB>();
    lds_barrier();
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      readA(0, 0, kk);
      readB(0, 0, kk);
    }
    wait_lgkmcnt0();
    if (!landed) wait_vmcnt<3 * JA + 2 * JB>();
    lds_barrier();

    // the copies awaited in the first five phases were requested before the previous tile's
    // stores, whose epilogue waited for them
    Sums acc;
    step(acc, I0{}, std::false_type{}, std::integral_constant<int, 4>{}, fullc, landed);
    step(acc, I1{}, std::false_type{}, I1{}, fullc, landed);
    for (int t = 2; t + 2 < KT; t += 2) {
      step(acc, I0{}, std::false_type{}, I0{}, fullc, false);
      step(acc, I1{}, std::false_type{}, I0{}, fullc, false);
    }
    request_from(nth_tile(n + 1), buf1, 0);   // (past the last tile: an earlier one again, not used)
    step(acc, I0{}, std::false_type{}, I0{}, fullc, false);
    step(acc, I1{}, std::true_type{}, I0{}, fullc, false);

    // ---- epilogue: acc * scale_a * scale_b (+ bias) in fp32, left to right, then one cast.
    // Each wave takes 32 rows x 64 columns (16-bit outputs; 32 columns of 4-byte ones) at a time
    // through its 4 KiB: rows of 128 bytes, chunk c at slot c ^ (row & 7), written out in whole
    // 128-byte lines, 8 rows a store, while the next 32 rows are computed.  The stores are buffer
    // stores, which drop what lies outside the problem and are issued whatever the mask: the wait
    // behind the first of them counts them.
    const int ln = fresh_lane();
    const int erow = ln & 31, ehalf = ln >> 5, srow = ln >> 3, sch = ln & 7;
    constexpr int FN = SILU ? QB : QN;                // output fragments across
    constexpr int ES = OD == I8L_F32 ? 4 : 2, EPC = 16 / ES;   // bytes of an element, elements of a chunk
    constexpr int FG = OD == I8L_F32 ? 1 : 2;         // fragments at a time
    constexpr int PER = FN < FG ? FN : FG;
    const int cw = wn * 32 * FN, nw = g0.col * BNO + cw;
    int8_t* stg = lds + STG + wave * 4096;
    const auto bufC = __builtin_amdgcn_make_buffer_rsrc((char*)p.out + (int64_t)g0.row0 * p.ldc * ES, 0,
                                                        0x7fffffff, 0x00020000);
    // the next tile's scales, and the source rows of the one after it
    const GroupTile g1 = nth_tile(n + 1), g2 = nth_tile(n + 2);
    const int td = 64 * wave + ln;
    const int src1 = td < BM ? sh.source[buf1][td] : -1;
    const int src2 = source_of(g2, td);
    const Operands next = operands_of(g1, src1, td);
    constexpr int NB = decltype(fullc)::value ? 2 * QA : QA;   // blocks of 32 rows
    // (every load is requested before the first store, so the wait behind the stores covers them)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int x0 = 0; x0 < FN; x0 += PER) {
      v4i pack[2][PER][OD == I8L_F32 ? 4 : 2];        // a block's values as stored, one ahead
      auto compute = [&](int b, v4i (&o)[PER][OD == I8L_F32 ? 4 : 2]) {
        const int h = b / QA, i = b % QA;
        const float sam = sh.sa[half][h * (BM / 2) + (wm * QA + i) * 32 + erow];
#pragma unroll
        for (int c = 0; c < PER; ++c)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int x = x0 + c, col = cw + 32 * x + 8 * q + 4 * ehalf;
            const float4 s0 = *(const float4*)&sh.sb[half][col];
            const float4 s1 = *(const float4*)&sh.sb[half][SILU ? BNO + col : col];
            float4 b0 = {}, b1 = {};
            if constexpr (BIAS) {
              b0 = *(const float4*)&sh.bias[half][col];
              b1 = *(const float4*)&sh.bias[half][SILU ? BNO + col : col];
            }
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              auto scaled = [&](int32_t a, const float4& s, const float4& b) {
                float y = (float)a;
                y = y * sam;
                y = y * (r == 0 ? s.x : r == 1 ? s.y : r == 2 ? s.z : s.w);
                if constexpr (BIAS) y = y + (r == 0 ? b.x : r == 1 ? b.y : r == 2 ? b.z : b.w);
                return y;
              };
              if constexpr (SILU)
                v[r] = silu_mul<OD == I8L_F32>(scaled(acc[h][0][i][x][4 * q + r], s0, b0),
                                               scaled(acc[h][1][i][x][4 * q + r], s1, b1));
              else
                v[r] = scaled(acc[h][x / QB][i][x % QB][4 * q + r], s0, b0);
              // the value itself is rounded to fp16 in a cast of its own: opaque, or the product
              // and the cast become one v_fma_mixlo_f16, which rounds once
              if constexpr (OD == I8L_F16) asm volatile("" : "+v"(v[r]));
            }
            if constexpr (OD == I8L_F32) {
              o[c][q] = __builtin_bit_cast(v4i, make_float4(v[0], v[1], v[2], v[3]));
            } else {
              o[c][q / 2][q % 2 * 2] = (int)f32x2_to_act2<OD>(v[0], v[1]);
              o[c][q / 2][q % 2 * 2 + 1] = (int)f32x2_to_act2<OD>(v[2], v[3]);
            }
          }
      };
      auto stage = [&](const v4i (&o)[PER][OD == I8L_F32 ? 4 : 2]) {
#pragma unroll
        for (int c = 0; c < PER; ++c)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (OD == I8L_F32)
              *(v4i*)(stg + erow * 128 + (((2 * q + ehalf) ^ (erow & 7)) * 16)) = o[c][q];
            else
              *(uint2*)(stg + erow * 128 + (((4 * c + q) ^ (erow & 7)) * 16) + 8 * ehalf) =
                  make_uint2((uint32_t)o[c][q / 2][q % 2 * 2], (uint32_t)o[c][q / 2][q % 2 * 2 + 1]);
          }
      };
      auto store = [&](int b) {
        const int row0 = b / QA * (BM / 2) + (wm * QA + b % QA) * 32;
        const int n = nw + 32 * x0 + EPC * sch;
        const bool in = n < width && sch * EPC < 32 * PER;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int row = 8 * y + srow;
          const v4i v = *(const v4i*)(stg + row * 128 + ((sch ^ srow) * 16));
          const uint32_t at = (uint32_t)(((row0 + row) * (int)p.ldc + n) * ES);
          __builtin_amdgcn_raw_buffer_store_b128(
              __builtin_bit_cast(v4u, v), bufC,
              in && row0 + row < rows ? at : kOutside, 0, kStoreCpol);
        }
      };
      compute(0, pack[0]);
      stage(pack[0]);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (b + 1 < NB) compute(b + 1, pack[(b + 1) % 2]);
        __builtin_amdgcn_sched_barrier(0);            // (else the registers of several blocks live at a time)
        store(b);
        if (b + 1 < NB) stage(pack[(b + 1) % 2]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (x0 == 0) {
        // the loads above and every copy in flight (the next tile's first two steps) have landed past
        // here, so the next tile's first waits need not count past this tile's stores
        asm volatile("" ::: "memory");
        wait_vmcnt<4 * NB>();
        asm volatile("" ::: "memory");
      }
    }
    keep(half ^ 1, src1, next, td);
    if (td < BM) sh.source[buf2][td] = src2;
    if (wave == 0 && (n + 1) % (kTiles / 2) == 0) find_tiles(n + 1 + kTiles / 2, kTiles / 2, ln);
  };
  // (the sums of the two kinds of tile never meet, so that each keeps its registers)
  for (int n = 0, tile = blockIdx.x; tile < tiles; ++n, tile += stride) {
    const GroupTile g = nth_tile(n);
    if (g.end - g.row0 > BM / 2) run_tile(std::true_type{}, g, n);
    else run_tile(std::false_type{}, g, n);
  }
}

// ------------------------------------------------------------------ host side
template <int WM, int QA, int QB, int OD, bool BIAS, bool SILU, bool STREAM>
hipError_t launch_k(const Grouped& p, hipStream_t st) {
  auto kern = grouped_phased<WM, QA, QB, OD, BIAS, SILU, STREAM>;
  constexpr int BM = WM * 64 * QA, BN = (4 / WM) * 64 * QB;
  constexpr size_t shm = 2 * (size_t)(BM + BN) * kStep + 4 * 4096 + sizeof(PhasedShared);
  static_assert(shm <= kMaxLds, "two buffers, the staging and the tables fit the LDS");
  static std::atomic<uint64_t> lds_done{0};  // devices this kernel is opted in on
  lds_opt_in((const void*)kern, shm, lds_done);
  const int width = SILU ? p.N / 2 : p.N, bno = SILU ? BN / 2 : BN;
  const int64_t tiles = most_blocks(p.R, p.E, BM) * ((width + bno - 1) / bno);
  const int grid = (int)std::min<int64_t>(tiles, cu_count() * (int)(kMaxLds / shm));
  // whole pairs of steps, the first and the last apart; zeros past K
  const int steps = std::max(4, 2 * ((p.K + 2 * kStep - 1) / (2 * kStep)));
  const uint32_t abytes = (uint32_t)((int64_t)(p.M - 1) * p.lda + p.K);
  const uint32_t bbytes = (uint32_t)((int64_t)(p.N - 1) * p.ldb + p.K);
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), shm, st, p, abytes, bbytes, steps);
  return hipGetLastError();
}

template <int WM, int QA, int QB, bool STREAM>
hipError_t launch_t(const Grouped& p, hipStream_t st) {
  auto go = [&](auto od) {
    constexpr int OD = decltype(od)::value;
    if (p.silu)
      return p.bias ? launch_k<WM, QA, QB, OD, true, true, STREAM>(p, st)
                    : launch_k<WM, QA, QB, OD, false, true, STREAM>(p, st);
    return p.bias ? launch_k<WM, QA, QB, OD, true, false, STREAM>(p, st)
                  : launch_k<WM, QA, QB, OD, false, false, STREAM>(p, st);
  };
  if (p.out_dtype == I8L_BF16) return go(std::integral_constant<int, I8L_BF16>{});
  if (p.out_dtype == I8L_F16) return go(std::integral_constant<int, I8L_F16>{});
  return go(std::integral_constant<int, I8L_F32>{});
}

}  // namespace

hipError_t launch_grouped_phased(int bm, bool stream, const Grouped& p, hipStream_t st) {
  if (bm == 64) return stream ? launch_t<1, 1, 1, true>(p, st) : launch_t<1, 1, 1, false>(p, st);
  if (bm == 128) return stream ? launch_t<2, 1, 2, true>(p, st) : launch_t<2, 1, 2, false>(p, st);
  return launch_t<2, 2, 2, false>(p, st);
}

}  // namespace i8l
