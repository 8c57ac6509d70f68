// The router of a layer with E experts: the k best experts of every token and their weights, and the
// order of the (token, choice) pairs by expert that the grouped products read.
//
//   picks      the k largest logits of a token, of equal ones the lower expert; one that is -inf or
//              NaN is never picked: expert -1, weight 0
//   weights    softmax: exp(x - max) over the sum of the picked (renormalize) or of all; sigmoid:
//              1 / (1 + exp(-x)), over the sum of the picked with renormalize; fp32
//   order      a stable counting sort of the pairs' flat index t * k + j by expert; pairs of no
//              expert (anything outside [0, E)) come last and are given place -1
//
// Selecting: 16 lanes a token, four tokens a wave, lane l holding the experts l * C .. l * C + C - 1 (one
// wide load).  The logits become unsigned keys in the same order; a pick is the largest key of the
// lanes (DPP within their row of 16), then the smallest expert that has it
// (which a 16-bit logit's key names itself).
//
// Ordering: up to 64 pairs by one wave, whose lanes compare their experts bit by bit with ballots; up
// to kOneGroup pairs (where experts are selected first, 64 tokens) in one workgroup and one launch: 256
// tokens of 8 given experts 5.0 us against 6.2 in two launches, 512 7.2 / 6.4; 64 tokens with their
// selection from 128 experts 7.2, 128 10.6 / 9.3.  More are cut into up to kChunks runs of tokens,
// one workgroup each: the first kernel selects and counts its run's pairs per expert, the second one
// adds up the runs before its own (all counts, from L2) and writes.  Within a run the waves take
// consecutive pieces, counted by LDS adds (sums of ones: any order) and then walked 64 pairs at a time,
// a pair's rank among equals from ballots of the expert's bits.  No atomic decides an order, so a call's
// results are the same every time.
//
// What bounds it is latency: 8192 tokens' 128 fp32 logits 7.2 us (8 rounds of dependent maxima, about 55
// instructions each for a wave's four tokens) and 5.8 for their order, each traced by itself, 11.9 for both in
// a row of passes, where a kernel starts under the end of the one before; one token's bf16 logits 3.9 us.
#include "i8l_common.h"

#include <algorithm>

namespace i8l {

namespace {

constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr int kMaxExperts = 512, kMaxPicks = 64;
constexpr int kSmall = 64;            // pairs that one wave orders
constexpr int64_t kOneGroup = 2048;   // pairs that one workgroup orders
constexpr int kChunks = 256;          // runs of tokens otherwise
constexpr int kMinRun = 4 * kWaves;   // tokens of a run at least: a round of the selecting waves

struct Route {
  const void* logits;       // NULL: `experts` are given
  int64_t ldl;
  float* weights;
  int32_t *experts, *offsets, *tokens, *places;
  int32_t* counts;          // [chunks][count_pitch(E)]
  int T, E, k, run, chunks; // run: tokens of a chunk
  int dtype, sigmoid, renormalize;
};

// Runs' counts are read four experts at a time.
__host__ __device__ constexpr int count_pitch(int E) { return (E + 1 + 3) & ~3; }

// Reductions over the 16 lanes of a DPP row; every lane returns its row's.
template <typename F>
__device__ __forceinline__ uint32_t row_reduce(uint32_t v, F f) {
  v = f(v, (uint32_t)dpp_i<kQuadSwap1>((int)v));
  v = f(v, (uint32_t)dpp_i<kQuadSwap2>((int)v));
  v = f(v, (uint32_t)dpp_i<kHalfMirror>((int)v));
  return f(v, (uint32_t)dpp_i<kRowMirror>((int)v));
}
__device__ __forceinline__ uint32_t row_umax(uint32_t v) {
  return row_reduce(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ uint32_t row_umin(uint32_t v) {
  return row_reduce(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
__device__ __forceinline__ float row_sum(float v) {
  return __uint_as_float(row_reduce(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// Keys in the order of the logits, 0 for -inf and NaN only; -0 counts as 0.  A 16-bit logit's key holds
// the expert too, the lower the larger, so that keys differ and the largest names its expert.
template <int DT>
__device__ __forceinline__ uint32_t key_of(uint32_t bits, int e) {
  if constexpr (DT == I8L_F32) {
    const float x = __uint_as_float(bits);
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x > -__builtin_inff() ? b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u) : 0u;
  } else {
    constexpr uint32_t inf = DT == I8L_BF16 ? 0x7f80u : 0x7c00u;
    const uint32_t b = bits == 0x8000u ? 0u : bits;
    const uint32_t u = b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
    return (b & 0x7fffu) > inf || b == (inf | 0x8000u) ? 0u : u << 16 | (0xffffu - e);
  }
}
template <int DT>
__device__ __forceinline__ float of_key(uint32_t key) {
  if constexpr (DT == I8L_F32)
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
  const uint32_t u = key >> 16;
  return act_to_f32<DT == I8L_F32 ? I8L_BF16 : DT>(u & 0x8000u ? u & 0x7fffu : ~u & 0xffffu);
}

// Logits [e0, e0 + C) of a row of E as keys, 0 past the last.  VEC: 16-byte aligned rows of whole
// vectors.
template <int C, int DT, bool VEC>
__device__ __forceinline__ void load_keys(const void* row, int e0, int E, uint32_t (&key)[C]) {
  if constexpr (VEC) {
    constexpr int V = DT == I8L_F32 ? 4 : 8;
#pragma unroll
    for (int c = 0; c < C; c += V) {
      const bool in = e0 + c < E;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (in) v = *(const uint4*)((const char*)row + (int64_t)(e0 + c) * (DT == I8L_F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t w = chunk_word(v, DT == I8L_F32 ? i : i / 2);
        const uint32_t x = DT == I8L_F32 ? w : i % 2 ? w >> 16 : w & 0xffffu;
        key[c + i] = in ? key_of<DT>(x, e0 + c + i) : 0u;
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      key[c] = 0;
      if (e0 + c < E)
        key[c] = key_of<DT>(DT == I8L_F32 ? ((const uint32_t*)row)[e0 + c] : ((const uint16_t*)row)[e0 + c],
                            e0 + c);
    }
  }
}

// exp(x - top) of the pickable; equal ones (both +inf among them) give 1
__device__ __forceinline__ float soft(float x, float top) {
  return x == top ? 1.0f : canon_expf(x - top);
}
__device__ __forceinline__ float sigmoid(float x) {
  const float z = canon_expf(-fabsf(x));
  return (x >= 0.0f ? 1.0f : z) / (1.0f + z);
}

// The picks of the tokens t0 .. t0 + 3 by one wave, 16 lanes each: lane l of 16 holds pick 16 s + l's
// expert in expert[s] (-1: none).  Tokens from t1 on: no picks, nothing written.
constexpr int kSlots = kMaxPicks / 16;
template <int C, int DT, bool VEC>
__device__ __forceinline__ void select(const Route& r, int t0, int t1, int lane, int (&expert)[kSlots]) {
  const int l = lane & 15, t = t0 + (lane >> 4);
  const bool in = t < t1;
  uint32_t key[C], mine[kSlots] = {};
  load_keys<C, DT, VEC>((const char*)r.logits + (in ? t : t0) * r.ldl * (DT == I8L_F32 ? 4 : 2), l * C,
                        r.E, key);
  float total = 0.0f;
  uint32_t top = key[0];
#pragma unroll
  for (int c = 1; c < C; ++c) top = max(top, key[c]);
  top = row_umax(top);
  const float tx = of_key<DT>(top);
  if (!r.renormalize && !r.sigmoid) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (key[c]) total += soft(of_key<DT>(key[c]), tx);
    total = row_sum(total);
  }
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    expert[s] = -1;
    for (int j = 16 * s; j < min(r.k, 16 * s + 16); ++j) {
      uint32_t best = key[0];
#pragma unroll
      for (int c = 1; c < C; ++c) best = max(best, key[c]);
      best = row_umax(best);
      uint32_t first = ~0u;
      if constexpr (DT == I8L_F32) {
#pragma unroll
        for (int c = C - 1; c >= 0; --c) first = key[c] == best ? l * C + c : first;
        first = row_umin(first);
#pragma unroll
        for (int c = 0; c < C; ++c) key[c] = first == l * C + c ? 0u : key[c];
      } else {
        first = 0xffffu - (best & 0xffffu);
#pragma unroll
        for (int c = 0; c < C; ++c) key[c] = key[c] == best ? 0u : key[c];
      }
      // (with nothing left to pick, best is 0)
      if (j == 16 * s + l && best) expert[s] = (int)first, mine[s] = best;
    }
  }
  float p[kSlots];
  float picked = 0.0f;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    p[s] = 0.0f;
    if (16 * s < r.k && expert[s] >= 0) {
      const float x = of_key<DT>(mine[s]);
      if (!r.sigmoid) p[s] = soft(x, tx);
      else if (!r.renormalize || tx >= 0.0f) p[s] = sigmoid(x);
      else p[s] = soft(x, tx) / (1.0f + canon_expf(x));   // over exp(max): the sum of any logits is not 0
    }
    picked += p[s];
  }
  if (r.renormalize) total = row_sum(picked);
  else if (r.sigmoid) total = 1.0f;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    if (!in) expert[s] = -1;
    if (in && 16 * s + l < r.k) {
      const int64_t at = (int64_t)t * r.k + 16 * s + l;
      r.weights[at] = total > 0.0f ? p[s] / total : 0.0f;
      r.experts[at] = expert[s];
    }
  }
}

__device__ __forceinline__ int bucket(int32_t e, int E) { return e >= 0 && e < E ? e : E; }

template <int W>
struct OrderShared {
  int32_t count[W][kMaxExperts + 1];       // of each wave's piece; then its next place
  int32_t before[kMaxExperts + 1];          // pairs of the expert in earlier runs
  int32_t total[kMaxExperts + 1];           // in all runs; then the expert's first place
};

// The order of one run, [t0, t1), whose experts are in memory.  counts: the runs' counts, or NULL
// where the run is all there is.
template <int W>
__device__ __forceinline__ void order_run(const Route& r, int chunk, int t0, int t1, OrderShared<W>& sh) {
  constexpr int kThreads = 64 * W;
  const int lane = threadIdx.x & 63, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int B = r.E + 1;
  const int i0 = t0 * r.k, n = (t1 - t0) * r.k;
  const int piece = ((n + W - 1) / W + 63) & ~63;
  const int w0 = min(wave * piece, n), w1 = min(w0 + piece, n);
  for (int b = lane; b < B; b += 64) sh.count[wave][b] = 0;
  if (r.chunks > 1)
    for (int b = tid; b < B; b += kThreads) sh.before[b] = sh.total[b] = 0;
  __syncthreads();
  for (int i = w0 + lane; i < w1; i += 64)
    atomicAdd(&sh.count[wave][bucket(r.experts[i0 + i], r.E)], 1);
  if (r.chunks > 1) {
    // the runs' counts, four experts a thread and several threads for them, each a share of the runs
    const int P = count_pitch(r.E) / 4, share = kThreads / P;
    if (tid < share * P) {
      const int b = tid % P * 4;
      int4 early = make_int4(0, 0, 0, 0), all = early;
#pragma unroll 8
      for (int c = tid / P; c < r.chunks; c += share) {
        const int4 v = *(const int4*)(r.counts + (int64_t)c * (4 * P) + b);
        all.x += v.x, all.y += v.y, all.z += v.z, all.w += v.w;
        if (c < chunk) early.x += v.x, early.y += v.y, early.z += v.z, early.w += v.w;
      }
      const int e[4] = {early.x, early.y, early.z, early.w}, a[4] = {all.x, all.y, all.z, all.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b + i < B) {
          atomicAdd(&sh.before[b + i], e[i]);
          atomicAdd(&sh.total[b + i], a[i]);
        }
    }
  }
  __syncthreads();
  if (r.chunks == 1)
    for (int b = tid; b < B; b += kThreads) {
      int v = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) v += sh.count[w][b];
      sh.total[b] = v;
      sh.before[b] = 0;
    }
  __syncthreads();
  if (wave == 0) {   // first places: an exclusive sum, a run of buckets a lane
    const int per = (B + 63) / 64, b0 = min(lane * per, B), b1 = min(b0 + per, B);
    int s = 0;
    for (int b = b0; b < b1; ++b) s += sh.total[b];
    int at = wave_scan(s) - s;
    for (int b = b0; b < b1; ++b) {
      const int v = sh.total[b];
      sh.total[b] = at;
      if (chunk == 0) r.offsets[b] = at;   // (bucket E starts where the last expert ends)
      at += v;
    }
  }
  __syncthreads();
  for (int b = tid; b < B; b += kThreads) {
    int at = sh.total[b] + sh.before[b];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int v = sh.count[w][b];
      sh.count[w][b] = at;
      at += v;
    }
  }
  __syncthreads();
  const int bits = 32 - __builtin_clz(r.E);
  volatile int32_t* next = sh.count[wave];
  for (int i = w0; i < w1; i += 64) {
    const bool in = i + lane < w1;
    const int b = in ? bucket(r.experts[i0 + i + lane], r.E) : -1;
    uint64_t same = __ballot(in);
    for (int x = 0; x < bits; ++x) {
      const uint64_t m = __ballot((b >> x) & 1);
      same &= (b >> x) & 1 ? m : ~m;
    }
    if (in) {
      const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
      const int place = next[b] + rank;
      const int flat = i0 + i + lane;
      r.places[flat] = b < r.E ? place : -1;
      r.tokens[place] = b < r.E ? flat / r.k : -1;
      __builtin_amdgcn_wave_barrier();
      if (rank == 0) next[b] = place + __popcll(same);   // (the first of its equals: place - 0)
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Up to kSmall pairs.  C = 0: experts are given.
template <int C, int DT, bool VEC>
__global__ void __launch_bounds__(256) moe_route_small(Route r) {
  __shared__ int32_t pair[kSmall], sorted[kSmall];
  const int tid = threadIdx.x, lane = tid & 63, n = r.T * r.k;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if constexpr (C > 0) {
    for (int t0 = 4 * wave; t0 < r.T; t0 += 16) {
      int expert[kSlots];
      select<C, DT, VEC>(r, t0, r.T, lane, expert);
      const int t = t0 + (lane >> 4);
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        const int j = 16 * s + (lane & 15);
        if (t < r.T && j < r.k) pair[t * r.k + j] = expert[s];
      }
    }
    __syncthreads();
  }
  if (wave == 0) {
    const bool in = lane < n;
    int b = 0x3ff;   // (past every expert: behind all)
    if (in) b = bucket(C > 0 ? pair[lane] : r.experts[lane], r.E);
    uint64_t less = 0, same = ~(uint64_t)0;
    for (int x = 9; x >= 0; --x) {
      const uint64_t m = __ballot((b >> x) & 1);
      if ((b >> x) & 1) less |= same & ~m, same &= m;
      else same &= ~m;
    }
    const int place = __popcll(less) + __popcll(same & (((uint64_t)1 << lane) - 1));
    sorted[place] = b;
    if (in) {
      r.places[lane] = b < r.E ? place : -1;
      r.tokens[place] = b < r.E ? lane / r.k : -1;
    }
  }
  __syncthreads();
  for (int e = tid; e <= r.E; e += 256) {   // pairs of experts below e
    int at = 0;
#pragma unroll
    for (int step = kSmall / 2; step; step /= 2)
      if (sorted[at + step - 1] < e) at += step;
    r.offsets[e] = at + (at == kSmall - 1 && sorted[at] < e);
  }
}
static_assert(kMaxExperts < 0x3ff, "the bits of an expert");

// The whole of a call that one workgroup takes.
template <int C, int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) moe_route_one(Route r) {
  __shared__ OrderShared<kWaves> sh;
  if constexpr (C > 0) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int expert[kSlots];
    for (int t = 4 * wave; t < r.T; t += 4 * kWaves) select<C, DT, VEC>(r, t, r.T, threadIdx.x & 63, expert);
    __syncthreads();   // the experts are in memory: order_run reads them from other waves
  }
  order_run(r, 0, 0, r.T, sh);
}

// A run's picks, and its pairs per expert.
template <int C, int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) moe_select(Route r) {
  __shared__ int32_t count[kMaxExperts + 1];
  const int t0 = blockIdx.x * r.run, t1 = min(t0 + r.run, r.T), lane = threadIdx.x & 63;
  for (int b = threadIdx.x; b <= r.E; b += kThreads) count[b] = 0;
  __syncthreads();
  if constexpr (C > 0) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int t = t0 + 4 * wave; t < t1; t += 4 * kWaves) {
      int expert[kSlots];
      select<C, DT, VEC>(r, t, t1, lane, expert);
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (t + (lane >> 4) < t1 && 16 * s + (lane & 15) < r.k)
          atomicAdd(&count[bucket(expert[s], r.E)], 1);
    }
  } else {
    for (int i = t0 * r.k + threadIdx.x; i < t1 * r.k; i += kThreads)
      atomicAdd(&count[bucket(r.experts[i], r.E)], 1);
  }
  __syncthreads();
  const int P = count_pitch(r.E);
  for (int b = threadIdx.x; b < P; b += kThreads)
    r.counts[(int64_t)blockIdx.x * P + b] = b <= r.E ? count[b] : 0;
}

// (eight waves: a run of 64 tokens of 8 picks is 64 pairs a wave)
constexpr int kOrderWaves = 8;
__global__ void __launch_bounds__(64 * kOrderWaves) moe_order(Route r) {
  __shared__ OrderShared<kOrderWaves> sh;
  const int t0 = blockIdx.x * r.run;
  order_run(r, blockIdx.x, t0, min(t0 + r.run, r.T), sh);
}

template <int C, int DT, bool VEC>
hipError_t launch_route(const Route& r, hipStream_t st) {
  if ((int64_t)r.T * r.k <= kSmall) {
    hipLaunchKernelGGL((moe_route_small<C, DT, VEC>), dim3(1), dim3(256), 0, st, r);
    return hipGetLastError();
  }
  if (r.chunks == 1) {
    hipLaunchKernelGGL((moe_route_one<C, DT, VEC>), dim3(1), dim3(kThreads), 0, st, r);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((moe_select<C, DT, VEC>), dim3(r.chunks), dim3(kThreads), 0, st, r);
  if (const hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL(moe_order, dim3(r.chunks), dim3(64 * kOrderWaves), 0, st, r);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_route_dt(const Route& r, hipStream_t st) {
  constexpr int V = DT == I8L_F32 ? 4 : 8;
  const bool vec = ((uintptr_t)r.logits & 15) == 0 && r.ldl % V == 0 && r.E % V == 0;
  auto go = [&](auto vc) {
    constexpr bool VEC = decltype(vc)::value;
    if (r.E <= 128) return launch_route<8, DT, VEC>(r, st);
    if (r.E <= 256) return launch_route<16, DT, VEC>(r, st);
    return launch_route<32, DT, VEC>(r, st);
  };
  return vec ? go(std::true_type{}) : go(std::false_type{});
}

// Tokens of a run and the number of runs.
void plan_runs(int64_t T, int64_t k, bool selects, int* run, int* chunks) {
  *run = (int)std::max<int64_t>(T, 1);
  *chunks = 1;
  if (T <= kMinRun || (!selects && T * k <= kOneGroup)) return;
  *run = (int)std::max<int64_t>(kMinRun, (T + kChunks - 1) / kChunks);
  *chunks = (int)((T + *run - 1) / *run);
}

int64_t workspace_bytes(int64_t T, int64_t E, int64_t k, bool selects) {
  if (T < 0 || E < 1 || k < 1 || E > kMaxExperts || k > kMaxPicks || T > ((int64_t)1 << 25) / k)
    return 0;
  int run, chunks;
  plan_runs(T, k, selects, &run, &chunks);
  return chunks > 1 ? (int64_t)chunks * count_pitch((int)E) * 4 : 0;
}

// The status of a call's sizes; -1 where they are fine.
int check_sizes(const char* who, int64_t T, int64_t E, int64_t k) {
  if (T < 0 || E < 1 || k < 1) {
    set_error("%s: bad sizes T=%lld E=%lld k=%lld", who, (long long)T, (long long)E, (long long)k);
    return I8L_INVALID_ARG;
  }
  if (E > kMaxExperts || k > kMaxPicks || T > ((int64_t)1 << 25) / k) {
    set_error("%s: up to %d experts, %d picks and 2^25 pairs, got T=%lld E=%lld k=%lld", who,
              kMaxExperts, kMaxPicks, (long long)T, (long long)E, (long long)k);
    return I8L_UNSUPPORTED;
  }
  return -1;
}

int run_route(const char* who, Route r, bool selects, int64_t T, int64_t E, int64_t k,
              void* workspace, int64_t bytes, hipStream_t st) {
  r.T = (int)T, r.E = (int)E, r.k = (int)k;
  plan_runs(T, k, selects, &r.run, &r.chunks);
  const int64_t need = workspace_bytes(T, E, k, selects);
  if (need > 0 && (!workspace || bytes < need || ((uintptr_t)workspace & 15))) {
    set_error("%s: a workspace of %lld bytes is needed, got %lld", who, (long long)need,
              (long long)(workspace ? bytes : 0));
    return I8L_INVALID_ARG;
  }
  r.counts = (int32_t*)workspace;
  hipError_t e;
  if (!r.logits) e = launch_route<0, I8L_F32, false>(r, st);
  else if (r.dtype == I8L_BF16) e = launch_route_dt<I8L_BF16>(r, st);
  else if (r.dtype == I8L_F16) e = launch_route_dt<I8L_F16>(r, st);
  else e = launch_route_dt<I8L_F32>(r, st);
  return hip_status(e, who);
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int64_t i8l_moe_route_workspace_bytes(int64_t T, int64_t E, int64_t k) {
  return workspace_bytes(T, E, k, true);
}

extern "C" int64_t i8l_moe_order_workspace_bytes(int64_t T, int64_t E, int64_t k) {
  return workspace_bytes(T, E, k, false);
}

extern "C" int i8l_moe_route(const void* logits, int64_t ldl, int32_t dtype, int64_t T, int64_t E,
                             int64_t k, int32_t scoring, int32_t renormalize, float* weights,
                             int32_t* experts, int32_t* offsets, int32_t* tokens, int32_t* places,
                             void* workspace, int64_t bytes, void* stream) {
  if (const int s = check_sizes("moe_route", T, E, k); s >= 0) return s;
  if (k > E || (T > 1 && ldl < E)) {
    set_error("moe_route: %lld picks of %lld experts, rows %lld apart", (long long)k, (long long)E,
              (long long)ldl);
    return I8L_INVALID_ARG;
  }
  if ((dtype != I8L_BF16 && dtype != I8L_F16 && dtype != I8L_F32) || scoring < 0 || scoring > 1) {
    set_error("moe_route: bf16, fp16 or fp32 logits, scoring 0 (softmax) or 1 (sigmoid)");
    return I8L_UNSUPPORTED;
  }
  if (!operands_ok("moe_route", {offsets}) ||
      (T > 0 && !operands_ok("moe_route", {logits, weights, experts, tokens, places})))
    return I8L_INVALID_ARG;
  Route r{logits, ldl, weights, experts, offsets, tokens, places};
  r.dtype = dtype, r.sigmoid = scoring, r.renormalize = renormalize != 0;
  return run_route("moe_route", r, true, T, E, k, workspace, bytes, (hipStream_t)stream);
}

extern "C" int i8l_moe_order(const int32_t* experts, int64_t T, int64_t E, int64_t k,
                             int32_t* offsets, int32_t* tokens, int32_t* places, void* workspace,
                             int64_t bytes, void* stream) {
  if (const int s = check_sizes("moe_order", T, E, k); s >= 0) return s;
  if (!operands_ok("moe_order", {offsets}) ||
      (T > 0 && !operands_ok("moe_order", {experts, tokens, places})))
    return I8L_INVALID_ARG;
  Route r{nullptr, 0, nullptr, const_cast<int32_t*>(experts), offsets, tokens, places};
  return run_route("moe_order", r, false, T, E, k, workspace, bytes, (hipStream_t)stream);
}
