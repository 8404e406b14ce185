// Log probabilities of given tokens, the entropy of their distributions and the most
// likely alternatives (kve_token_logprobs). The reference decodes greedily and scores
// nothing (kvengine/decode.py:57-332).
//
// The mathematics. With m the row's maximum, S = sum e^(x - m) and T = sum (x - m) e^(x - m):
// log p(t) = x[t] - m - log S, entropy = -sum p log p = log S - T / S. T is never positive,
// so nothing cancels in the entropy. Exponents are taken in base 2, y = (x - m) log2(e);
// y is held above -1000, where 2^y is 0, so that an id of no mass (-inf, a mask) adds
// 0 * 2^y to T and not a NaN.
//
// Launches: chunks of 2048 logits, a wave each, leave (m, S, T) and the maxima of their
// groups of consecutive ids (16 lanes' vectors: 128 ids in bf16, 64 in fp32); then a
// workgroup per row joins the chunks in 64 bits and finds the alternatives. Ids are ranked
// by logit, equal ones lowest first. The n likeliest ids lie in the n groups whose maxima
// rank first (an id of another group has n group maxima before it), so the row is read
// again in those groups alone.
//
// What bounds it, at 151936 ids in bf16. 160 rows and 20 alternatives: statistics 13.5 us (3.6
// TB/s), the row's workgroup 10, two selections one after another with their dependent reads
// (84 us in all with the largest taken n times). One row: 3.5 and 7.8, launches and round trips.

#include "kve_logits.h"

#include <algorithm>
#include <cmath>

namespace kve {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 32;

struct LogprobArgs {
  const void* logits;
  int64_t stride;  // elements between rows
  const int32_t* tokens;
  int rows, V, chunks, top;
  float *logprobs, *entropy;
  int32_t* top_ids;
  float* top_logprobs;
  float4* stats;      // [rows][chunks]: m, S, T
  uint32_t* groups;   // [rows][chunks * groups of a chunk]: order_key of the maximum
};

constexpr float kLog2e = 1.44269504088896340736f;

// Ids of a group: a 16-byte vector of each of 16 lanes.
template <typename E>
constexpr int kGroup = 16 * kVec<E>;
template <typename E>
constexpr int kChunkGroups = kChunk / kGroup<E>;

template <typename E>
__global__ __launch_bounds__(kThreads) void logprob_stats_kernel(LogprobArgs a) {
  constexpr int N = Piece<E>::N, NV = Piece<E>::NV;
  const int l = threadIdx.x & 63;
  const int total = a.rows * a.chunks, step = gridDim.x * kWaves;
  int i = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= total) return;
  Piece<E> t;
  const auto load = [&](int at) {
    const int r = at / a.chunks;
    t.load(static_cast<const E*>(a.logits) + r * a.stride, at - r * a.chunks, l, a.V);
  };
  load(i);
  for (;;) {
    Piece<E> x = t;
    const int next = i + step;
    if (next < total) load(next);
    float f[NV * N], g[NV], m = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int e = 0; e < N; ++e) f[v * N + e] = logit<E>(x.x[v], e);
      g[v] = f[v * N];
#pragma unroll
      for (int e = 1; e < N; ++e) g[v] = max_nan(g[v], f[v * N + e]);
#pragma unroll
      for (int e = 0; e < N; ++e) lo = fminf(lo, f[v * N + e]);
    }
    if (a.top) {
      // the 16 lanes' maxima of each vector; lane v of them keeps the v-th, for one store
#pragma unroll
      for (int v = 0; v < NV; ++v) g[v] = row_max(g[v]);
      float mine = g[0];
#pragma unroll
      for (int v = 1; v < NV; ++v) mine = (l & 15) == v ? g[v] : mine;
      if ((l & 15) < NV)
        a.groups[static_cast<size_t>(i) * kChunkGroups<E> + (l & 15) * 4 + (l >> 4)] = order_key(mine + 0.0f);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) m = max_nan(m, g[v]);
    m = wave_max(m);
    float s = 0.0f, w = 0.0f;
    if (__all(lo > -1e30f) && fabsf(m) < 1000.0f) {
      // y = x log2(e) - k in one rounding, k = m log2(e) rounded; what that lost, d, is made
      // good on the sums
      const float k = m * kLog2e, d = fmaf(m, kLog2e, -k);
#pragma unroll
      for (int e = 0; e < NV * N; ++e) {
        const float y = fmaf(f[e], kLog2e, -k);
        const float p = __builtin_amdgcn_exp2f(y);
        s += p;
        w = fmaf(y, p, w);
      }
      s = wave_sum(s);
      w = wave_sum(w);
      const float r = __builtin_amdgcn_exp2f(-d);
      w = (w - d * s) * r;
      s *= r;
    } else {
      // any values: an id of no mass adds nothing to w; the difference comes first, for a
      // maximum at the type's lowest value times log2(e) is -inf
      const float c = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int e = 0; e < NV * N; ++e) {
        const float y = max_nan((f[e] - c) * kLog2e, -1000.0f);
        const float p = __builtin_amdgcn_exp2f(y);
        s += p;
        w = fmaf(y, p, w);
      }
      s = wave_sum(s);
      w = wave_sum(w);
    }
    if (l == 0) a.stats[i] = float4{m, s, w, 0.0f};
    if (next >= total) return;
    i = next;
  }
}

// Reductions of 64-bit values over the 16 lanes of a row, by moves inside the vector unit
// (swap neighbours, swap pairs, mirror halves, mirror the row).
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_mov64(uint64_t u) {
  const uint32_t lo = static_cast<uint32_t>(u), hi = static_cast<uint32_t>(u >> 32);
  return static_cast<uint64_t>(static_cast<uint32_t>(
             __builtin_amdgcn_mov_dpp(static_cast<int>(hi), CTRL, 0xf, 0xf, false))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(lo), CTRL, 0xf, 0xf, false));
}
template <typename Op>
__device__ __forceinline__ uint64_t row_reduce64(uint64_t v, Op op) {
  v = op(v, dpp_mov64<0xB1>(v));
  v = op(v, dpp_mov64<0x4E>(v));
  v = op(v, dpp_mov64<0x141>(v));
  return op(v, dpp_mov64<0x140>(v));
}
__device__ __forceinline__ double row_add(double v) {
  return __builtin_bit_cast(
      double, row_reduce64(__builtin_bit_cast(uint64_t, v), [](uint64_t a, uint64_t b) {
        return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b));
      }));
}

// A key ranks a value by itself, then by its place: the later the smaller.
__device__ __forceinline__ uint64_t rank_key(uint32_t order, int place) {
  return static_cast<uint64_t>(order) << 32 | ~static_cast<uint32_t>(place);
}
__device__ __forceinline__ int place_of(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

// The n largest of `count` keys by a workgroup: found(i, key) for i = 0 .. n - 1 (n <= kMaxTop
// of them are not 0, which stands for none). 16 threads' keys are a set, 64 sets; the n-th
// largest of the sets' maxima is no larger than the n-th largest key, so only what reaches
// it (n and a few more where the keys lie at random) is listed and ranked by counting. Where
// the list does not hold that, the largest is taken n times. key(i): key i.
constexpr int kFinishThreads = 1024;
constexpr int kList = 1024;
struct Select {
  alignas(16) uint64_t sets[64], list[kList];
  uint64_t least;
  int listed;
};

// keys of sm[0, count) above `mine`, count even
__device__ __forceinline__ int keys_above(const uint64_t* sm, int count, uint64_t mine) {
  int above = 0;
#pragma unroll 16
  for (int q = 0; q < count; q += 2) {
    const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(sm + q);
    above += (k.x > mine) + (k.y > mine);
  }
  return above;
}

template <typename K, typename F>
__device__ __forceinline__ void select_largest(Select& sm, int n, int count, int tid, K key, F found) {
  constexpr int KEEP = 4;  // keys a thread holds on to: 4096 in all
  uint64_t held[KEEP], set = 0;
#pragma unroll
  for (int e = 0; e < KEEP; ++e) held[e] = key(min(tid + e * kFinishThreads, count - 1));
#pragma unroll
  for (int e = 0; e < KEEP; ++e) {
    held[e] = tid + e * kFinishThreads < count ? held[e] : 0;
    set = umax64(set, held[e]);
  }
  const auto each = [&](auto put) {
#pragma unroll
    for (int e = 0; e < KEEP; ++e) put(held[e]);
    for (int i0 = KEEP * kFinishThreads; i0 < count; i0 += kFinishThreads)
      put(i0 + tid < count ? key(i0 + tid) : 0);
  };
  if (count > KEEP * kFinishThreads) each([&](uint64_t k) { set = umax64(set, k); });
  set = row_reduce64(set, umax64);
  if ((tid & 15) == 0) sm.sets[tid >> 4] = set;
  if (tid == 0) {
    sm.listed = 0;
    sm.least = 1;  // fewer than n sets hold anything: every key reaches it
  }
  __syncthreads();
  if (tid < 64) {
    const uint64_t mine = sm.sets[tid];
    if (keys_above(sm.sets, 64, mine) == n - 1 && mine) sm.least = mine;
  }
  __syncthreads();
  const uint64_t least = sm.least;
  // a wave counts what it will list, takes that many places and fills them
  int places = 0;
  each([&](uint64_t k) { places += __popcll(__ballot(k >= least)); });
  if (places) {
    int at = 0;
    if ((tid & 63) == 0) at = atomicAdd(&sm.listed, places);
    at = __builtin_amdgcn_readfirstlane(at);
    each([&](uint64_t k) {
      const uint64_t here = __ballot(k >= least);
      if (!here) return;
      const int x = at + __popcll(here & ((1ull << (tid & 63)) - 1));
      if (k >= least && x < kList) sm.list[x] = k;
      at += __popcll(here);
    });
  }
  __syncthreads();
  const int listed = sm.listed;
  if (listed <= kList) {
    if (tid == 0 && listed < kList) sm.list[listed] = 0;
    __syncthreads();
    if (tid < listed) {
      const uint64_t mine = sm.list[tid];
      const int above = keys_above(sm.list, (listed + 1) & ~1, mine);
      if (above < n) found(above, mine);
    }
  } else {
    uint64_t under = ~0ull;  // (also the key of a NaN at place 0: the first turn takes any)
    for (int x = 0; x < n; ++x) {
      uint64_t best = 0;
      for (int i = tid; i < count; i += kFinishThreads) {
        const uint64_t k = key(i);
        if (x == 0 || k < under) best = umax64(best, k);
      }
      best = max_across_groups_u64(row_reduce64(best, umax64));
      __syncthreads();
      if ((tid & 63) == 0) sm.sets[tid >> 6] = best;
      __syncthreads();
      under = sm.sets[0];
      for (int q = 1; q < kFinishThreads / 64; ++q) under = umax64(under, sm.sets[q]);
      if (tid == 0) found(x, under);
    }
  }
  __syncthreads();
}

template <typename E>
__global__ __launch_bounds__(kFinishThreads) void logprob_finish_kernel(LogprobArgs a) {
  constexpr double kLn2 = 0.69314718055994530942;
  constexpr int kFinishWaves = kFinishThreads / 64;
  __shared__ double sm_s[kFinishThreads / 16], sm_t[kFinishThreads / 16];
  __shared__ float sm_m[kFinishWaves];
  __shared__ int sm_groups[kMaxTop];
  __shared__ Select sm_select;
  const int r = blockIdx.x, tid = threadIdx.x;
  const E* row = static_cast<const E*>(a.logits) + r * a.stride;
  const float4* st = a.stats + static_cast<size_t>(r) * a.chunks;
  const int t = a.tokens[r];
  const bool inside = t >= 0 && t < a.V;
  const float given = to_f32(row[inside ? t : 0]);
  // every thread's first chunk stays in registers: 1024 are a vocabulary of 2097152
  const float4 none = {-INFINITY, 0.0f, 0.0f, 0.0f};
  const float4 own = tid < a.chunks ? st[tid] : none;
  float M = own.x;
  for (int c = tid + kFinishThreads; c < a.chunks; c += kFinishThreads) M = max_nan(M, st[c].x);
  M = wave_max(M);
  if ((tid & 63) == 0) sm_m[tid >> 6] = M;
  __syncthreads();
  M = sm_m[0];
#pragma unroll
  for (int q = 1; q < kFinishWaves; ++q) M = max_nan(M, sm_m[q]);
  double S = 0.0, T = 0.0;
  const auto join = [&](const float4& p) {
    if (p.x == -INFINITY) return;  // no mass
    const double d = (static_cast<double>(p.x) - M) * static_cast<double>(kLog2e);
    const float f = __builtin_amdgcn_exp2f(static_cast<float>(d));
    S += static_cast<double>(f) * p.y;
    if (f != 0.0f) T += f * (p.z + d * p.y);
  };
  join(own);
  for (int c = tid + kFinishThreads; c < a.chunks; c += kFinishThreads) join(st[c]);
  S = row_add(S);
  T = row_add(T);
  if ((tid & 15) == 0) {
    sm_s[tid >> 4] = S;
    sm_t[tid >> 4] = T;
  }
  __syncthreads();
  // 64 rows' sums, four to a lane of 16
  S = row_add((sm_s[tid & 15] + sm_s[16 + (tid & 15)]) + (sm_s[32 + (tid & 15)] + sm_s[48 + (tid & 15)]));
  T = row_add((sm_t[tid & 15] + sm_t[16 + (tid & 15)]) + (sm_t[32 + (tid & 15)] + sm_t[48 + (tid & 15)]));
  const double logS = log(S);  // a row of no mass: -inf, and NaN below
  // (M off first: beside a maximum of 3e38 log S would be lost)
  const auto logprob = [&](float x) {
    return static_cast<float>(static_cast<double>(x) - M - logS);
  };
  if (tid == 0) {
    a.logprobs[r] = inside ? logprob(given) : NAN;
    a.entropy[r] = static_cast<float>(logS - kLn2 * T / S);
  }
  if (!a.top) return;
  // the groups of the likeliest ids, then the ids: one code for both
  const int G = cdiv(a.V, kGroup<E>), groups = min(a.top, G);
  const uint32_t* gk = a.groups + static_cast<size_t>(r) * a.chunks * kChunkGroups<E>;
#pragma unroll 1
  for (int ids = 0; ids < 2; ++ids) {
    select_largest(
        sm_select, ids ? a.top : groups, ids ? groups * kGroup<E> : G, tid,
        [&](int i) -> uint64_t {
          if (!ids) return rank_key(gk[i], i);
          const int id = sm_groups[i / kGroup<E>] * kGroup<E> + i % kGroup<E>;
          const E x = row[min(id, a.V - 1)];
          return id < a.V ? rank_key(order_key(to_f32(x) + 0.0f), id) : 0;
        },
        [&](int n, uint64_t key) {
          if (!ids) {
            sm_groups[n] = place_of(key);
            return;
          }
          const size_t at = static_cast<size_t>(r) * a.top + n;
          a.top_ids[at] = place_of(key);
          // the logit, out of the order it was ranked by
          a.top_logprobs[at] = logprob(unorder_key(static_cast<uint32_t>(key >> 32)));
        });
  }
}

// Workgroups of the stats launch: 8 per compute unit.
constexpr int kStatGrid = 2048;

struct LogprobCfg {
  int chunks;
  size_t groups, bytes;
};

static LogprobCfg logprob_cfg(int rows, int V, int top, int dtype) {
  LogprobCfg c{};
  c.chunks = cdiv(V, kChunk);
  const size_t parts = static_cast<size_t>(rows) * c.chunks;
  c.groups = parts * sizeof(float4);
  const int per = dtype == KVE_DTYPE_BF16 ? kChunkGroups<uint16_t> : kChunkGroups<float>;
  c.bytes = c.groups + (top ? parts * per * sizeof(uint32_t) : 0);
  return c;
}

template <typename E>
static void launch_logprobs(const LogprobArgs& a, hipStream_t st) {
  // every wave the same number of chunks
  const int total = a.rows * a.chunks, each = cdiv(total, kStatGrid * kWaves);
  hipLaunchKernelGGL(logprob_stats_kernel<E>, dim3(cdiv(total, each * kWaves)), dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(logprob_finish_kernel<E>, dim3(a.rows), dim3(kFinishThreads), 0, st, a);
}

}  // namespace kve

using namespace kve;

extern "C" size_t kve_logprobs_workspace_bytes(int rows, int vocab, int top, int dtype) {
  if (rows <= 0 || vocab <= 0 || vocab > (1 << 30) || top < 0 || top > kMaxTop ||
      (dtype != KVE_DTYPE_BF16 && dtype != KVE_DTYPE_F32))
    return 0;
  return logprob_cfg(rows, vocab, top, dtype).bytes;
}

extern "C" int kve_token_logprobs(const void* logits, int64_t row_stride, const int32_t* tokens,
                                  int rows, int vocab, int top, int dtype, float* logprobs,
                                  float* entropy, int32_t* top_ids, float* top_logprobs,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (rows == 0) return KVE_OK;
  KVE_REQUIRE(logits && tokens && logprobs && entropy && (top == 0 || (top_ids && top_logprobs)),
              "kve_token_logprobs: null pointer argument");
  KVE_REQUIRE(rows > 0 && vocab > 0 && vocab <= (1 << 30) && top >= 0 && top <= kMaxTop && top <= vocab,
              "kve_token_logprobs: %d rows of %d, %d alternatives (at most %d)", rows, vocab, top,
              kMaxTop);
  KVE_REQUIRE(dtype == KVE_DTYPE_BF16 || dtype == KVE_DTYPE_F32, "kve_token_logprobs: dtype %d",
              dtype);
  const size_t esz = dtype == KVE_DTYPE_BF16 ? 2 : 4;
  KVE_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (esz - 1)) == 0,
              "kve_token_logprobs: logits are not aligned to their type");
  const LogprobCfg c = logprob_cfg(rows, vocab, top, dtype);
  // (chunks are counted in 32 bits, and a launch has below 2^32 threads)
  KVE_REQUIRE(rows < (1 << 22) && static_cast<long long>(rows) * c.chunks < (1ll << 30),
              "kve_token_logprobs: %d rows of %d too large for one launch", rows, vocab);
  KVE_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              "kve_token_logprobs: workspace required (16-byte aligned)");
  if (workspace_bytes < c.bytes) {
    set_error("kve_token_logprobs: workspace %zu bytes, need %zu", workspace_bytes, c.bytes);
    return KVE_EWORKSPACE;
  }
  LogprobArgs a{};
  a.logits = logits;
  a.stride = row_stride;
  a.tokens = tokens;
  a.rows = rows;
  a.V = vocab;
  a.chunks = c.chunks;
  a.top = top;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.stats = static_cast<float4*>(workspace);
  a.groups = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + c.groups);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == KVE_DTYPE_BF16) launch_logprobs<uint16_t>(a, st);
  else launch_logprobs<float>(a, st);
  return check_launch("kve_token_logprobs");
}
