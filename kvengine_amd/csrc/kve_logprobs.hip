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
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float g = logit<E>(x.x[v], 0);
#pragma unroll
      for (int e = 1; e < N; ++e) g = max_nan(g, logit<E>(x.x[v], e));
      if (a.top) {
        g = row_max(g);
        if ((l & 15) == 0)
          a.groups[static_cast<size_t>(i) * kChunkGroups<E> + v * 4 + (l >> 4)] = order_key(g + 0.0f);
      }
      m = max_nan(m, g);
    }
    m = wave_max(m);
    // (the difference first: a maximum at the type's lowest value times log2(e) is -inf)
    const float mc = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, w = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      x.hide(v);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float y = max_nan((logit<E>(x.x[v], e) - mc) * kLog2e, -1000.0f);
        const float p = __builtin_amdgcn_exp2f(y);
        s += p;
        w = fmaf(y, p, w);
      }
    }
    s = wave_sum(s);
    w = wave_sum(w);
    if (l == 0) a.stats[i] = float4{m, s, w, 0.0f};
    if (next >= total) return;
    i = next;
  }
}

// The largest key of the workgroup below `under`, keys held by the threads; every
// thread gets it. sm: 2 * kWaves, halves used in turn so that one barrier is enough.
__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* sm, int tid) {
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) v = umax64(v, __shfl_xor(v, o));
  v = max_across_groups_u64(v);
  if ((tid & 63) == 0) sm[tid >> 6] = v;
  __syncthreads();
  v = sm[0];
#pragma unroll
  for (int q = 1; q < kWaves; ++q) v = umax64(v, sm[q]);
  return v;
}

__device__ __forceinline__ double block_sum(double v, double* sm, int tid) {
  v = wave_sum64(v);
  if ((tid & 63) == 0) sm[tid >> 6] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) t += sm[q];
  __syncthreads();
  return t;
}

template <typename E>
__global__ __launch_bounds__(kThreads) void logprob_finish_kernel(LogprobArgs a) {
  constexpr double kLn2 = 0.69314718055994530942;
  __shared__ double sm_d[kWaves];
  __shared__ float sm_m[kWaves];
  __shared__ uint64_t sm_k[2 * kWaves];
  __shared__ int sm_groups[kMaxTop];
  const int r = blockIdx.x, tid = threadIdx.x;
  const E* row = static_cast<const E*>(a.logits) + r * a.stride;
  const float4* st = a.stats + static_cast<size_t>(r) * a.chunks;
  float M = -INFINITY;
  for (int c = tid; c < a.chunks; c += kThreads) M = max_nan(M, st[c].x);
  M = wave_max(M);
  if ((tid & 63) == 0) sm_m[tid >> 6] = M;
  __syncthreads();
  M = sm_m[0];
#pragma unroll
  for (int q = 1; q < kWaves; ++q) M = max_nan(M, sm_m[q]);
  double S = 0.0, T = 0.0;
  for (int c = tid; c < a.chunks; c += kThreads) {
    const float4 p = st[c];
    if (p.x == -INFINITY) continue;  // no mass
    const double d = (static_cast<double>(p.x) - M) * static_cast<double>(kLog2e);
    const double f = exp2(d);
    S += f * p.y;
    if (f > 0.0) T += f * (p.z + d * p.y);
  }
  S = block_sum(S, sm_d, tid);
  T = block_sum(T, sm_d, tid);
  const double logS = log(S);  // a row of no mass: -inf, and NaN below
  // (M off first: beside a maximum of 3e38 log S would be lost)
  const auto logprob = [&](E x) {
    return static_cast<float>(static_cast<double>(to_f32(x)) - M - logS);
  };
  if (tid == 0) {
    const int t = a.tokens[r];
    a.logprobs[r] = t >= 0 && t < a.V ? logprob(row[t]) : NAN;
    a.entropy[r] = static_cast<float>(logS - kLn2 * T / S);
  }
  if (!a.top) return;
  // the groups of the likeliest ids
  const int G = cdiv(a.V, kGroup<E>), ng = min(a.top, G);
  const uint32_t* gk = a.groups + static_cast<size_t>(r) * a.chunks * kChunkGroups<E>;
  uint64_t under = ~0ull;
  for (int n = 0; n < ng; ++n) {
    uint64_t best = 0;
    for (int g = tid; g < G; g += kThreads) {
      const uint64_t k = static_cast<uint64_t>(gk[g]) << 32 | ~static_cast<uint32_t>(g);
      if (k < under) best = umax64(best, k);
    }
    under = block_max(best, sm_k + (n & 1) * kWaves, tid);
    if (tid == 0) sm_groups[n] = static_cast<int>(~static_cast<uint32_t>(under));
  }
  __syncthreads();
  under = ~0ull;
  for (int n = 0; n < a.top; ++n) {
    uint64_t best = 0;
    for (int c = tid; c < ng * kGroup<E>; c += kThreads) {
      const int id = sm_groups[c / kGroup<E>] * kGroup<E> + c % kGroup<E>;
      if (id >= a.V) continue;
      const uint64_t k = static_cast<uint64_t>(order_key(to_f32(row[id]) + 0.0f)) << 32 |
                         ~static_cast<uint32_t>(id);
      if (k < under) best = umax64(best, k);
    }
    under = block_max(best, sm_k + (n & 1) * kWaves, tid);
    if (tid == 0) {
      const int id = static_cast<int>(~static_cast<uint32_t>(under));
      a.top_ids[static_cast<size_t>(r) * a.top + n] = id;
      a.top_logprobs[static_cast<size_t>(r) * a.top + n] = logprob(row[id]);
    }
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
  hipLaunchKernelGGL(logprob_stats_kernel<E>, dim3(std::min(kStatGrid, cdiv(a.rows * a.chunks, kWaves))),
                     dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(logprob_finish_kernel<E>, dim3(a.rows), dim3(kThreads), 0, st, a);
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
  KVE_REQUIRE(static_cast<long long>(rows) * c.chunks < (1ll << 30),
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
