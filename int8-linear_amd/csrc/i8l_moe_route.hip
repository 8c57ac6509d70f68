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
// Selecting: a wave a token, lane l holding the experts l, l + 64, ...  The logits become unsigned
// keys in the same order, so a pick is one maximum over the wave (DPP) and a compare of every
// register against it, whose first set lane is the lowest expert; all of that is uniform.
//
// Ordering: up to kOneGroup pairs in one workgroup and one launch.  More are cut into up to kChunks
// runs of tokens, one workgroup each: the first kernel selects and counts its run's pairs per
// expert, the second one adds up the runs before its own (kChunks * E counts, from L2) and writes.
// Within a run the waves take consecutive pieces, counted by LDS adds (sums of ones: any order) and
// then walked 64 pairs at a time, a pair's rank among equals from ballots of the expert's bits.  No
// atomic decides an order, so a call's results are the same every time.
#include "i8l_common.h"

#include <algorithm>

namespace i8l {

namespace {

constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr int kMaxExperts = 512, kMaxPicks = 64;
constexpr int64_t kOneGroup = 1024;   // pairs that one workgroup orders in the selecting launch
constexpr int kChunks = 128;          // runs of tokens otherwise
constexpr int kMinRun = 32;           // tokens of a run at least

struct Route {
  const void* logits;       // NULL: `experts` are given
  int64_t ldl;
  float* weights;
  int32_t *experts, *offsets, *tokens, *places;
  int32_t* counts;          // [chunks][E + 1]
  int T, E, k, run, chunks; // run: tokens of a chunk
  int dtype, sigmoid, renormalize;
};

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = max(v, (uint32_t)dpp_i<kQuadSwap1>((int)v));
  v = max(v, (uint32_t)dpp_i<kQuadSwap2>((int)v));
  v = max(v, (uint32_t)dpp_i<kHalfMirror>((int)v));
  v = max(v, (uint32_t)dpp_i<kRowMirror>((int)v));
  const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)v, 0),
                         (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
  const uint32_t b = max((uint32_t)__builtin_amdgcn_readlane((int)v, 32),
                         (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
  return max(a, b);
}

__device__ __forceinline__ float wave_sum(float v) {
  v = v + __int_as_float(dpp_i<kQuadSwap1>(__float_as_int(v)));
  v = v + __int_as_float(dpp_i<kQuadSwap2>(__float_as_int(v)));
  v = v + __int_as_float(dpp_i<kHalfMirror>(__float_as_int(v)));
  v = v + __int_as_float(dpp_i<kRowMirror>(__float_as_int(v)));
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    s[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16 * i));
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// Keys in the order of the floats, never 0 for a number; 0 for -inf and NaN.  (-0 counts as 0.)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t u = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return x > -__builtin_inff() ? u : 0u;
}
__device__ __forceinline__ float of_key(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

template <int DT>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (DT == I8L_F32) return ((const float*)p)[i];
  else return act_to_f32<DT>(((const uint16_t*)p)[i]);
}

// exp(x - top) of the pickable; equal ones (both +inf among them) give 1
__device__ __forceinline__ float soft(float x, float top) {
  return x == top ? 1.0f : canon_expf(x - top);
}
__device__ __forceinline__ float sigmoid(float x) {
  const float z = canon_expf(-fabsf(x));
  return (x >= 0.0f ? 1.0f : z) / (1.0f + z);
}

// The picks of token t by one wave: lane j < k holds pick j's expert (-1: none).
template <int C, int DT>
__device__ __forceinline__ int select(const Route& r, int64_t t, int lane) {
  uint32_t key[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int e = 64 * c + lane;
    key[c] = e < r.E ? key_of(load_logit<DT>(r.logits, t * r.ldl + e)) : 0u;
  }
  uint32_t all[C];
#pragma unroll
  for (int c = 0; c < C; ++c) all[c] = key[c];
  int expert = -1;
  uint32_t mine = 0, top = 0;
  for (int j = 0; j < r.k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int c = 1; c < C; ++c) best = max(best, key[c]);
    best = wave_umax(best);
    if (best == 0) break;   // nothing left to pick
    if (j == 0) top = best;
    int at = 0, first = 0;
#pragma unroll
    for (int c = C - 1; c >= 0; --c) {
      const uint64_t m = __ballot(key[c] == best);
      if (m) at = c, first = __builtin_ctzll(m);
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c == at && lane == first) key[c] = 0;
    if (lane == j) expert = 64 * at + first, mine = best;
  }
  const float tx = of_key(top);
  float p = 0.0f, total = 0.0f;
  if (expert >= 0) {
    const float x = of_key(mine);
    if (!r.sigmoid) p = soft(x, tx);
    else if (!r.renormalize || tx >= 0.0f) p = sigmoid(x);
    else p = soft(x, tx) / (1.0f + canon_expf(x));   // over exp(max): the sum of any logits is not 0
  }
  if (r.renormalize) {
    total = wave_sum(p);
  } else if (!r.sigmoid) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (all[c]) total += soft(of_key(all[c]), tx);
    total = wave_sum(total);
  } else {
    total = 1.0f;
  }
  if (lane < r.k) {
    const int64_t at = t * r.k + lane;
    r.weights[at] = total > 0.0f ? p / total : 0.0f;
    r.experts[at] = expert;
  }
  return expert;
}

__device__ __forceinline__ int bucket(int32_t e, int E) { return e >= 0 && e < E ? e : E; }

struct OrderShared {
  int32_t count[kWaves][kMaxExperts + 1];   // of each wave's piece; then its next place
  int32_t before[kMaxExperts + 1];          // pairs of the expert in earlier runs
  int32_t total[kMaxExperts + 1];           // in all runs; then the expert's first place
};

// The order of one run, [t0, t1), whose experts are in memory.  counts: the runs' counts, or NULL
// where the run is all there is.
__device__ __forceinline__ void order_run(const Route& r, int chunk, int t0, int t1, OrderShared& sh) {
  const int lane = threadIdx.x & 63, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int B = r.E + 1;
  const int i0 = t0 * r.k, n = (t1 - t0) * r.k;
  const int piece = ((n + kWaves - 1) / kWaves + 63) & ~63;
  const int w0 = min(wave * piece, n), w1 = min(w0 + piece, n);
  for (int b = lane; b < B; b += 64) sh.count[wave][b] = 0;
  if (r.chunks > 1)
    for (int b = tid; b < B; b += kThreads) sh.before[b] = sh.total[b] = 0;
  __syncthreads();
  for (int i = w0 + lane; i < w1; i += 64)
    atomicAdd(&sh.count[wave][bucket(r.experts[i0 + i], r.E)], 1);
  if (r.chunks > 1) {
    // the runs' counts, several threads an expert, each a share of the runs
    const int share = max(1, kThreads / B);
    for (int x = tid; x < share * B; x += kThreads) {
      const int b = x % B;
      int early = 0, all = 0;
#pragma unroll 8
      for (int c = x / B; c < r.chunks; c += share) {
        const int v = r.counts[c * B + b];
        all += v;
        early += c < chunk ? v : 0;
      }
      atomicAdd(&sh.before[b], early);
      atomicAdd(&sh.total[b], all);
    }
  }
  __syncthreads();
  if (r.chunks == 1)
    for (int b = tid; b < B; b += kThreads) {
      int v = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v += sh.count[w][b];
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
    for (int w = 0; w < kWaves; ++w) {
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

template <int C, int DT>
__device__ __forceinline__ void select_run(const Route& r, int t0, int t1) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int t = t0 + wave; t < t1; t += kWaves) select<C, DT>(r, t, threadIdx.x & 63);
}

// The whole of a small call.  C = 0: experts are given.
template <int C, int DT>
__global__ void __launch_bounds__(kThreads) moe_route_one(Route r) {
  __shared__ OrderShared sh;
  if constexpr (C > 0) {
    select_run<C, DT>(r, 0, r.T);
    __syncthreads();   // the experts are in memory: order_run reads them from other waves
  }
  order_run(r, 0, 0, r.T, sh);
}

// A run's picks, and its pairs per expert.
template <int C, int DT>
__global__ void __launch_bounds__(kThreads) moe_select(Route r) {
  __shared__ int32_t count[kMaxExperts + 1];
  const int t0 = blockIdx.x * r.run, t1 = min(t0 + r.run, r.T), lane = threadIdx.x & 63;
  for (int b = threadIdx.x; b <= r.E; b += kThreads) count[b] = 0;
  __syncthreads();
  if constexpr (C > 0) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int t = t0 + wave; t < t1; t += kWaves) {
      const int e = select<C, DT>(r, t, lane);
      if (lane < r.k) atomicAdd(&count[bucket(e, r.E)], 1);
    }
  } else {
    for (int i = t0 * r.k + threadIdx.x; i < t1 * r.k; i += kThreads)
      atomicAdd(&count[bucket(r.experts[i], r.E)], 1);
  }
  __syncthreads();
  for (int b = threadIdx.x; b <= r.E; b += kThreads)
    r.counts[(int64_t)blockIdx.x * (r.E + 1) + b] = count[b];
}

__global__ void __launch_bounds__(kThreads) moe_order(Route r) {
  __shared__ OrderShared sh;
  const int t0 = blockIdx.x * r.run;
  order_run(r, blockIdx.x, t0, min(t0 + r.run, r.T), sh);
}

template <int C, int DT>
hipError_t launch_route(const Route& r, hipStream_t st) {
  if (r.chunks == 1) {
    hipLaunchKernelGGL((moe_route_one<C, DT>), dim3(1), dim3(kThreads), 0, st, r);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((moe_select<C, DT>), dim3(r.chunks), dim3(kThreads), 0, st, r);
  if (const hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL(moe_order, dim3(r.chunks), dim3(kThreads), 0, st, r);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_route_dt(const Route& r, hipStream_t st) {
  if (r.E <= 64) return launch_route<1, DT>(r, st);
  if (r.E <= 128) return launch_route<2, DT>(r, st);
  if (r.E <= 256) return launch_route<4, DT>(r, st);
  return launch_route<8, DT>(r, st);
}

// Tokens of a run and the number of runs.
void plan_runs(int64_t T, int64_t k, int* run, int* chunks) {
  *run = (int)std::max<int64_t>(T, 1);
  *chunks = 1;
  if (T * k <= kOneGroup) return;
  *run = (int)std::max<int64_t>(kMinRun, (T + kChunks - 1) / kChunks);
  *chunks = (int)((T + *run - 1) / *run);
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

int run_route(const char* who, Route r, int64_t T, int64_t E, int64_t k, void* workspace,
              int64_t workspace_bytes, hipStream_t st) {
  r.T = (int)T, r.E = (int)E, r.k = (int)k;
  plan_runs(T, k, &r.run, &r.chunks);
  const int64_t need = i8l_moe_order_workspace_bytes(T, E, k);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 3))) {
    set_error("%s: a workspace of %lld bytes is needed, got %lld", who, (long long)need,
              (long long)(workspace ? workspace_bytes : 0));
    return I8L_INVALID_ARG;
  }
  r.counts = (int32_t*)workspace;
  hipError_t e;
  if (!r.logits) e = launch_route<0, I8L_F32>(r, st);
  else if (r.dtype == I8L_BF16) e = launch_route_dt<I8L_BF16>(r, st);
  else if (r.dtype == I8L_F16) e = launch_route_dt<I8L_F16>(r, st);
  else e = launch_route_dt<I8L_F32>(r, st);
  return hip_status(e, who);
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int64_t i8l_moe_order_workspace_bytes(int64_t T, int64_t E, int64_t k) {
  if (T < 0 || E < 1 || k < 1 || E > kMaxExperts || k > kMaxPicks || T > ((int64_t)1 << 25) / k)
    return 0;
  int run, chunks;
  plan_runs(T, k, &run, &chunks);
  return chunks > 1 ? (int64_t)chunks * (E + 1) * 4 : 0;
}

extern "C" int i8l_moe_route(const void* logits, int64_t ldl, int32_t dtype, int64_t T, int64_t E,
                             int64_t k, int32_t scoring, int32_t renormalize, float* weights,
                             int32_t* experts, int32_t* offsets, int32_t* tokens, int32_t* places,
                             void* workspace, int64_t workspace_bytes, void* stream) {
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
  return run_route("moe_route", r, T, E, k, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int i8l_moe_order(const int32_t* experts, int64_t T, int64_t E, int64_t k,
                             int32_t* offsets, int32_t* tokens, int32_t* places, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (const int s = check_sizes("moe_order", T, E, k); s >= 0) return s;
  if (!operands_ok("moe_order", {offsets}) ||
      (T > 0 && !operands_ok("moe_order", {experts, tokens, places})))
    return I8L_INVALID_ARG;
  Route r{nullptr, 0, nullptr, const_cast<int32_t*>(experts), offsets, tokens, places};
  return run_route("moe_order", r, T, E, k, workspace, workspace_bytes, (hipStream_t)stream);
}
