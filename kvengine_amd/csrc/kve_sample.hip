// Verification of drafted tokens by rejection sampling from given uniform numbers
// (kve_sample_verify; the sampled counterpart of the greedy accept of
// kvengine/speculative.py:169-197).
//
// The mathematics. p = softmax(target / T), q = softmax(draft / T) at each drafted
// position; draft x stands while u q(x) < p(x). At the first that falls the token is
// drawn from r = max(p - q, 0), else, after the last draft, from p, by inversion: the
// lowest id whose running sum exceeds u * sum(r).
//
// The draw is in 64 bits. The drawn id is a place among up to 150 000 running sums, and an
// error in a sum moves the draws whose place falls between its two values. 400000 draws of
// 151936 ids of spread 3 (T = 0.7, 0.8, 1; on the CPU) differ from the definition's in 8 to
// 32 of a hundred with 32-bit sums one after another, in 1 to 3 of a thousand with 32-bit
// sums by chunks of 2048, and still in 0.5 to 4 of 10^4 with 64-bit sums of 32-bit weights.
// Weights within e of theirs move at most about 2 V e: these (4e-14) one draw in 10^8. A
// weight costs a wave 86 cycles in 64 bits and 22 in 32 bits (its logit's loads 35, at the
// chip's copy rate), so only the logits of the position that decides are taken in 64 bits:
// which position that is follows from 32-bit sums, whose error is known, and where a test
// lies within it (2 in 10^5 tests) from that row's 64-bit ones.
//
// Launches, each a dependency of the next over the whole vocabulary; a chunk is 2048
// logits, one per wave:
//  stats   every (row, chunk): maximum, and the sum of 2^((l - max) c) in 32 bits,
//          c = log2(e) / T. Without drafts (k = 0) there is no test, and it is the
//          64-bit sum that the draw takes.
//  rest    every (sequence, chunk), k > 0: the rows' chunks joined, the tests, and at the
//          deciding position the chunk's 64-bit sums
//  pick    every sequence: the exact ratio of the two rows' sums, the chunk that holds
//          the drawn place, then its ids
// The stats launch reads all logits once and bounds the call; the others re-read one
// position's rows, and one chunk.
//
// The rest without its own pass over the vocabulary. With e = 2^((target - mp) c), g the
// draft's and L = sum(e) / sum(g), r is max(e - L g, 0) / sum(e). L is only known after
// a pass, but to 2^-16 from the 32-bit sums (L'). So the pass sums e - L' g over the ids
// where it is positive, and g over the same ids: the rest is the first minus (L - L')
// times the second. An id where |e - L' g| <= 2^-16 L' g may be on either side. Those are
// summed apart, with the least and the largest e / g among them: L above all of them
// leaves them out, below all of them takes them in, and only a chunk with L between them
// is summed again by `pick`. In bf16 logits t - d takes few values, so that where L is
// near one's e / g nearly every chunk has ids there, all of one e / g: re-summing those 75
// chunks took one call in three of 32 sequences 145 us for 44.

#include "kve_common.h"

#include <algorithm>
#include <type_traits>

namespace kve {

// The deciding position of a sequence.
struct SamplePick {
  double lam;       // L' above; drafts with probabilities, not all accepted
  float mp, mq;     // row maxima of the target and the draft
  int n_acc, skip;  // skip: id left out (a rejected draft without a distribution), or -1
};

// What `rest` leaves of a chunk at the deciding position.
struct RestSums {
  double e, g;      // sums over the chunk
  double over, gp;  // sum of e - L' g over the ids where it is positive, and of their g;
                    // without a draft's distribution: sum of e without `skip`, 0
  double eu, gu;    // sums of e and g over the undecided ids
  double lo, hi;    // the least and the largest e / g of those (none: inf, -inf; nothing
                    // known: -inf, inf)
  // for L the undecided ids are all out, all in, or the chunk is to be summed again
  // (also where L is as near to them as 64-bit weights are apart)
  __device__ __forceinline__ bool out(double lam) const { return lam >= hi; }
  __device__ __forceinline__ bool in(double lam) const { return lam < lo * (1.0 - 0x1p-40); }
  __device__ __forceinline__ bool marked(double lam) const { return !out(lam) && !in(lam); }
};

struct SampleArgs {
  const void *target, *draft;
  int64_t ts, tp, ds, dp;  // element strides per sequence and position
  const int32_t* drafts;
  const float *u_accept, *u_sample, *temps;
  double temp;
  const int32_t *lens, *seq_rows;
  int num_rows, B, k, V, rows, chunks;  // rows per sequence: k + 1 target, then k draft
  int32_t *n_acc, *emitted, *keep;
  double* sums;    // [B][rows][chunks]: sum of the chunk relative to its maximum
  float* maxes;    // [B][rows][chunks]
  RestSums* rest;  // [B][chunks]
  SamplePick* picks;  // [B]
};

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kChunk = 2048;  // logits: 32 per lane of a wave, 8 per thread of a workgroup

// log2(e) / T, or 0 where T is not positive and finite (the sequence has no answer). T in 32
// bits would move every weight by up to 3e-8 (l - max) / T of it: 2 to 3 draws in 10^4 of
// 151936 ids at T = 0.7 and 0.8, which are no 32-bit numbers.
__device__ __forceinline__ double sample_rate(const SampleArgs& a, int b) {
  const double t = a.temps ? a.temps[b] : a.temp;
  return t > 0.0 && t < INFINITY ? 1.4426950408889634074 / t : 0.0;
}

// 2^y = 2^n 2^f with n = round(y), f = y - n: 1 + f q(f), q the polynomial of degree 8
// that meets (2^f - 1) / f at the nine Chebyshev points of [-1/2, 1/2]. Within 4e-14
// of 2^f, and 2^0 is 1 exactly, so that equal logits give exactly equal sums.
__device__ __forceinline__ double exp2_poly(double f) {
  double p = 1.0203121063391729e-07;
  p = fma(p, f, 1.3255224878668817e-06);
  p = fma(p, f, 1.525268684626772e-05);
  p = fma(p, f, 0.00015403455852453838);
  p = fma(p, f, 0.0013333558179043112);
  p = fma(p, f, 0.009618129159402558);
  p = fma(p, f, 0.055504108664760424);
  p = fma(p, f, 0.2402265069581299);
  p = fma(p, f, 0.6931471805599453);
  return fma(p, f, 1.0);
}

// The weight 2^((l - m) c) of a logit against a maximum m (center() of it), for every
// value: 0 where it underflows and at -inf, NaN where l or m is NaN or m is +inf.
__device__ __forceinline__ double weight(float l, double m, double rate) {
  // the product rounded on its own: an exponent far below any is then a whole number,
  // where a fused y - round(y) would be the product's rounding error, which may be large
#pragma clang fp contract(off)
  const double y = (static_cast<double>(l) - m) * rate;
  const double n = __builtin_rint(y);
  const double w = __builtin_amdgcn_ldexp(exp2_poly(y - n), static_cast<int>(fmax(n, -4096.0)));
  return l == -INFINITY ? 0.0 : w;
}

// The same where (l - m) c is known to lie in [kNear, 0]: the rounding and the power of
// two come from adding 1.5 * 2^52, whose low word then holds n, in place of the slower
// rounding, conversion and scaling instructions.
constexpr double kNear = -1000.0;
__device__ __forceinline__ double weight_near(float l, double m, double rate) {
  constexpr double kShift = 6755399441055744.0;
  const double d = static_cast<double>(l) - m;
  const double t = fma(d, rate, kShift);
  const double p = exp2_poly(fma(d, rate, kShift - t));
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}

__device__ __forceinline__ bool is_near(float l, double m, double rate) {
  return (static_cast<double>(l) - m) * rate >= kNear;  // (false for a NaN)
}

// What weights are taken against: a maximum of -inf (no mass) counts as 0.
__device__ __forceinline__ double center(float m) {
  return m == -INFINITY ? 0.0 : static_cast<double>(m);
}

// (v_maximum / v_minimum: a NaN stays, so that it reaches the sums)
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }

// over the 16 lanes of a row
__device__ __forceinline__ float row_max(float v) {
  v = max_nan(v, dpp_mov<0xB1>(v));
  v = max_nan(v, dpp_mov<0x4E>(v));
  v = max_nan(v, dpp_mov<0x141>(v));
  return max_nan(v, dpp_mov<0x140>(v));
}
__device__ __forceinline__ double row_sum(double v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  v = row_max(v);
  const uint32_t u = __float_as_uint(v);
  const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = max_nan(__uint_as_float(h[0]), __uint_as_float(h[1]));
  const uint32_t w = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return max_nan(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v = row_sum(v);
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

template <typename E>
__device__ __forceinline__ float to_f32(E v) {
  if constexpr (std::is_same_v<E, float>) return v;
  else return bf16_to_f32(v);
}

template <typename E>
constexpr int kVec = 16 / sizeof(E);

// A 16-byte vector of logits as stored, from element i0 on, of a row of V; those past the
// end are -inf. Rows may start at any element (an odd vocabulary): gfx950 reads vectors
// at the type's alignment.
template <typename E>
__device__ __forceinline__ u32x4 load_raw(const E* row, int i0, int V) {
  constexpr int N = kVec<E>;
  struct __attribute__((packed, aligned(sizeof(E)))) Vec { u32x4 v; };
  if (i0 + N <= V) return reinterpret_cast<const Vec*>(row + i0)->v;
  u32x4 x;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (N == 4) {
      x[w] = i0 + w < V ? __float_as_uint(row[i0 + w]) : 0xff800000u;
    } else {
      const uint32_t lo = i0 + 2 * w < V ? row[i0 + 2 * w] : 0xff80u;
      const uint32_t hi = i0 + 2 * w + 1 < V ? row[i0 + 2 * w + 1] : 0xff80u;
      x[w] = lo | hi << 16;
    }
  }
  return x;
}

// Logit e of such a vector.
template <typename E>
__device__ __forceinline__ float logit(const u32x4& x, int e) {
  if constexpr (kVec<E> == 4) return __uint_as_float(x[e]);
  else return __uint_as_float(e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16);
}

template <typename E>
__device__ __forceinline__ void load_logits(const E* row, int i0, int V, float (&x)[kVec<E>]) {
  const u32x4 raw = load_raw<E>(row, i0, V);
#pragma unroll
  for (int e = 0; e < kVec<E>; ++e) x[e] = logit<E>(raw, e);
}

template <typename E>
__device__ __forceinline__ const E* logits_row(const SampleArgs& a, int b, int r) {
  return r <= a.k ? static_cast<const E*>(a.target) + b * a.ts + r * a.tp
                  : static_cast<const E*>(a.draft) + b * a.ds + (r - a.k - 1) * a.dp;
}

// A lane's share of a chunk as stored: logits ch * kChunk + v * 64 * N + lane * N ...
template <typename E>
struct Piece {
  static constexpr int N = kVec<E>, NV = kChunk / (64 * N);
  u32x4 x[NV];
  __device__ __forceinline__ void load(const E* row, int ch, int l, int V) {
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v] = load_raw<E>(row, (ch * NV + v) * 64 * N + l * N, V);
  }
  // Vector v from here on only: without it the compiler converts every logit of the
  // chunk ahead of the sums (120 registers, four waves a SIMD).
  __device__ __forceinline__ void hide(int v) { __asm__ volatile("" : "+v"(x[v])); }
};

// Every wave takes chunks (sequences x rows x chunks, chunks fastest) wave, wave +
// waves of the grid, ..., the next one loading while one is summed.
template <typename E, bool WIDE>
__global__ __launch_bounds__(kThreads) void sample_stats_kernel(SampleArgs a) {
  constexpr int N = Piece<E>::N, NV = Piece<E>::NV;
  const int l = threadIdx.x & 63;
  const int total = a.B * a.rows * a.chunks, step = gridDim.x * kWaves;
  int i = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= total) return;
  Piece<E> t;
  int b = 0;
  const auto load = [&](int at) {
    const int br = at / a.chunks;
    b = br / a.rows;
    t.load(logits_row<E>(a, b, br - b * a.rows), at - br * a.chunks, l, a.V);
  };
  load(i);
  for (;;) {
    Piece<E> x = t;
    const double rate = sample_rate(a, b);
    const int next = i + step;
    if (next < total) load(next);
    float m = logit<E>(x.x[0], 0), lo = m;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        m = max_nan(m, logit<E>(x.x[v], e));
        if (WIDE) lo = min_nan(lo, logit<E>(x.x[v], e));
      }
    }
    m = wave_max(m);
    double s = 0.0;
    if constexpr (WIDE) {
      const double c = center(m);
      if (__all(is_near(lo, c, rate))) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          x.hide(v);
#pragma unroll
          for (int e = 0; e < N; ++e) s += weight_near(logit<E>(x.x[v], e), c, rate);
        }
      } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          x.hide(v);
#pragma unroll
          for (int e = 0; e < N; ++e) s += weight(logit<E>(x.x[v], e), c, rate);
        }
      }
    } else {
      // 32 bits: an exponent y is off by 3 roundings of it and 2^y by its instruction's, so
      // the sum by 2^-23 (2 + 1.1 mean|y|), mean |y| being at most log2 of the vocabulary
      // (an entropy) and a bit, and by a rounding of each of a lane's 32 additions:
      // below 5e-6 of it (kMargin)
      const float c = m == -INFINITY ? 0.0f : m, f = static_cast<float>(rate);
      float p = 0.0f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int e = 0; e < N; ++e) p += __builtin_amdgcn_exp2f((logit<E>(x.x[v], e) - c) * f);
      }
      s = p;
    }
    s = wave_sum64(s);
    if (l == 0) {
      a.maxes[i] = m;
      a.sums[i] = s;
    }
    if (next >= total) return;
    i = next;
  }
}

// A chunk's sum against its row's maximum (center mc) instead of its own. A chunk of no
// mass holds 0, one with a NaN in it that.
__device__ __forceinline__ double chunk_sum(double s, float m, double mc, double rate) {
  return m == -INFINITY ? s : s * weight(m, mc, rate);
}

// Sum of a value over the workgroup's threads, to each of them.
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

// How far apart u q and p (from 32-bit sums, relative to p) decide a test, and e and
// L' g an id's sign: more than the two sums, 5e-6 each, can be off (1e-5).
constexpr double kMargin = 1.0 / 65536;

// The deciding position of sequence b, by a whole workgroup: every row's chunks joined
// (16 lanes a row), then the drafts' tests, a draft per thread; the lowest that fails
// decides. sm_s: rows doubles, then rows floats.
template <typename E>
__device__ __forceinline__ SamplePick decide(const SampleArgs& a, int b, double rate, double* sm_s,
                                             double* sm, int* sm_first) {
  float* sm_m = reinterpret_cast<float*>(sm_s + a.rows);
  const int tid = threadIdx.x, l16 = tid & 15;
  // the drafts' logits, asked for before the statistics arrive
  int x = -1;
  float lp = 0, lq = 0;
  double u = 0;
  if (tid < a.k) {
    x = a.drafts[static_cast<size_t>(b) * a.k + tid];
    u = a.u_accept[static_cast<size_t>(b) * a.k + tid];
    if (x >= 0 && x < a.V) {
      lp = to_f32(logits_row<E>(a, b, tid)[x]);
      if (a.draft) lq = to_f32(logits_row<E>(a, b, a.k + 1 + tid)[x]);
    }
  }
  for (int r = tid >> 4; r < a.rows; r += kThreads / 16) {
    const size_t at = (static_cast<size_t>(b) * a.rows + r) * a.chunks;
    // the lanes' first chunks stay in registers: 80 are a vocabulary of 163840
    constexpr int KEEP = 5;
    float m[KEEP], M = -INFINITY;
    double s[KEEP], S = 0.0;
#pragma unroll
    for (int q = 0; q < KEEP; ++q) {
      const int c = q * 16 + l16;
      m[q] = c < a.chunks ? a.maxes[at + c] : -INFINITY;
      s[q] = c < a.chunks ? a.sums[at + c] : 0.0;
      M = max_nan(M, m[q]);
    }
    for (int c = KEEP * 16 + l16; c < a.chunks; c += 16) M = max_nan(M, a.maxes[at + c]);
    M = row_max(M);
    const double mc = center(M);
#pragma unroll
    for (int q = 0; q < KEEP; ++q) S += chunk_sum(s[q], m[q], mc, rate);
    for (int c = KEEP * 16 + l16; c < a.chunks; c += 16)
      S += chunk_sum(a.sums[at + c], a.maxes[at + c], mc, rate);
    S = row_sum(S);
    if (l16 == 0) {
      sm_s[r] = S;
      sm_m[r] = M;
    }
  }
  __syncthreads();
  // 0: stands, 1: falls (a NaN too), 2: too near for 32-bit sums. Temperatures whose
  // exponents leave 32 bits are always too near.
  int state = 0;
  const int rp = tid, rq = a.k + 1 + tid;
  if (tid < a.k) {
    state = 1;
    if (x >= 0 && x < a.V) {
      const double p = weight(lp, center(sm_m[rp]), rate) / sm_s[rp];
      const double q = a.draft ? weight(lq, center(sm_m[rq]), rate) / sm_s[rq] : 1.0;
      const bool coarse = !(rate > 1e-30 && rate < 1e30);
      if (p > 0.0 && (coarse || fabs(u * q - p) <= kMargin * p)) state = 2;
      else if (u * q < p) state = 0;
      if (coarse) state = 2;
    }
  }
  for (;;) {
    if (tid == 0) *sm_first = 2 * a.k;
    __syncthreads();
    if (tid < a.k && state) atomicMin(sm_first, 2 * tid + (state == 2));
    __syncthreads();
    const int first = *sm_first;
    __syncthreads();
    if (!(first & 1)) break;
    // the test in 64 bits: the two rows summed by this workgroup
    const int j = first >> 1;
    const auto row_sum64 = [&](int r) {
      const E* row = logits_row<E>(a, b, r);
      const double mc = center(sm_m[r]);
      double s = 0.0;
      for (int i0 = tid * kVec<E>; i0 < a.V; i0 += kThreads * kVec<E>) {
        float y[kVec<E>];
        load_logits<E>(row, i0, a.V, y);
#pragma unroll
        for (int e = 0; e < kVec<E>; ++e) s += weight(y[e], mc, rate);
      }
      return block_sum(s, sm, tid);
    };
    const double sp = row_sum64(j), sq = a.draft ? row_sum64(a.k + 1 + j) : 1.0;
    if (tid == j) {
      const double p = weight(lp, center(sm_m[rp]), rate) / sp;
      const double q = a.draft ? weight(lq, center(sm_m[rq]), rate) / sq : 1.0;
      state = u * q < p ? 0 : 1;
    }
  }
  const int j = *sm_first >> 1;
  const bool both = a.draft && j < a.k;
  SamplePick p;
  p.n_acc = j;
  p.mp = sm_m[j];
  p.mq = both ? sm_m[a.k + 1 + j] : 0.0f;
  p.lam = both ? sm_s[j] / sm_s[a.k + 1 + j] : 0.0;
  p.skip = !a.draft && j < a.k ? a.drafts[static_cast<size_t>(b) * a.k + j] : -1;
  return p;
}

// Grid: sequences x groups of kWaves chunks, a chunk per wave.
template <typename E>
__global__ __launch_bounds__(kThreads) void sample_rest_kernel(SampleArgs a) {
  constexpr int N = Piece<E>::N, NV = Piece<E>::NV;
  extern __shared__ double sm_rows[];
  __shared__ double sm[kWaves];
  __shared__ int sm_first;
  const int l = threadIdx.x & 63, groups = cdiv(a.chunks, kWaves);
  const int b = blockIdx.x / groups;
  const int ch = (blockIdx.x - b * groups) * kWaves + (threadIdx.x >> 6);
  const double rate = sample_rate(a, b);
  if (!(rate > 0.0)) return;  // no answer: sample_pick_kernel says so without any sums
  const SamplePick p = decide<E>(a, b, rate, sm_rows, sm, &sm_first);
  if (ch == 0 && l == 0) a.picks[b] = p;
  if (ch >= a.chunks) return;
  const bool both = a.draft && p.n_acc < a.k;
  const double mp = center(p.mp), mq = center(p.mq);
  Piece<E> x, y;
  x.load(logits_row<E>(a, b, p.n_acc), ch, l, a.V);
  if (both) y.load(logits_row<E>(a, b, a.k + 1 + p.n_acc), ch, l, a.V);
  else y = x;
  float lo_p = INFINITY, lo_q = INFINITY;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      lo_p = min_nan(lo_p, logit<E>(x.x[v], e));
      lo_q = min_nan(lo_q, logit<E>(y.x[v], e));
    }
  }
  RestSums r{0.0, 0.0, 0.0, 0.0, 0.0, 0.0, INFINITY, -INFINITY};
  bool undecided = false;
  const double edge = kMargin * p.lam;
  const auto sum_both = [&](auto&& w) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      x.hide(v);
      y.hide(v);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double we = w(logit<E>(x.x[v], e), mp), wg = w(logit<E>(y.x[v], e), mq);
        const double d = we - p.lam * wg;
        r.e += we;
        r.g += wg;
        undecided |= wg > 0.0 && !(fabs(d) > edge * wg);
        r.over += d > 0.0 ? d : 0.0;
        r.gp += d > 0.0 ? wg : 0.0;
      }
    }
  };
  // The chunk once more, from memory and in a rolled loop (from the registers its weights
  // took 256 of them, and every chunk's pass 25 us for 17).
  const auto sum_apart = [&]() {
    const E *tr = logits_row<E>(a, b, p.n_acc), *dr = logits_row<E>(a, b, a.k + 1 + p.n_acc);
    r.over = r.gp = 0.0;
#pragma unroll 1
    for (int v = 0; v < NV; ++v) {
      const int i0 = (ch * NV + v) * 64 * N + l * N;
      const u32x4 xv = load_raw<E>(tr, i0, a.V), yv = load_raw<E>(dr, i0, a.V);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double we = weight(logit<E>(xv, e), mp, rate), wg = weight(logit<E>(yv, e), mq, rate);
        const double d = we - p.lam * wg;
        if (wg > 0.0 && !(fabs(d) > edge * wg)) {
          const double ratio = we / wg;
          r.eu += we;
          r.gu += wg;
          r.lo = fmin(r.lo, ratio);
          r.hi = fmax(r.hi, ratio);
        } else if (d > 0.0) {
          r.over += d;
          r.gp += wg;
        }
      }
    }
    r.eu = wave_sum64(r.eu);
    r.gu = wave_sum64(r.gu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      r.lo = fmin(r.lo, __shfl_xor(r.lo, o));
      r.hi = fmax(r.hi, __shfl_xor(r.hi, o));
    }
  };
  const auto sum_one = [&](auto&& w) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      x.hide(v);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double we = w(logit<E>(x.x[v], e), mp);
        r.e += we;
        r.over += (ch * NV + v) * 64 * N + l * N + e == p.skip ? 0.0 : we;
      }
    }
  };
  const auto near = [&](float t, double m) { return weight_near(t, m, rate); };
  const auto any = [&](float t, double m) { return weight(t, m, rate); };
  if (both) {
    if (__all(is_near(lo_p, mp, rate) && is_near(lo_q, mq, rate))) sum_both(near);
    else sum_both(any);
    if (!(p.lam > 0.0 && p.lam < INFINITY)) {  // no number to test against
      r.lo = -INFINITY;
      r.hi = INFINITY;
    } else if (__any(undecided)) {
      sum_apart();
    }
    r.g = wave_sum64(r.g);
    r.gp = wave_sum64(r.gp);
  } else {
    if (__all(is_near(lo_p, mp, rate))) sum_one(near);
    else sum_one(any);
  }
  r.e = wave_sum64(r.e);
  r.over = wave_sum64(r.over);
  if (l == 0) a.rest[static_cast<size_t>(b) * a.chunks + ch] = r;
}

// Exclusive prefix of a value over the workgroup's threads, and the total.
__device__ __forceinline__ double block_prefix(double v, double* sm, int tid, double& total) {
  const int l = tid & 63, w = tid >> 6;
  double inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(inc, o);
    if (l >= o) inc += up;
  }
  if (l == 63) sm[w] = inc;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) {
    if (q == w) before = total;
    total += sm[q];
  }
  __syncthreads();
  return before + inc - v;
}

// Grid: sequences. Thread t holds the sums of `per` consecutive chunks (one up to a
// vocabulary of 524288).
template <typename E>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs a) {
  constexpr int N = kVec<E>, NV = kChunk / (kThreads * N);  // a thread's ids are consecutive
  __shared__ double sm[kWaves], sm_ahead;
  __shared__ float sm_max[kWaves];
  __shared__ uint64_t sm_marked[kWaves];
  __shared__ int sm_at, sm_last;
  const int tid = threadIdx.x, w = tid >> 6, b = blockIdx.x;
  const double rate = sample_rate(a, b), u = a.u_sample[b];
  const auto answer = [&](int n_acc, int32_t token) {
    for (int j = tid; j <= a.k; j += kThreads) {
      const int32_t d = j < a.k ? a.drafts[static_cast<size_t>(b) * a.k + j] : -1;
      a.emitted[static_cast<size_t>(b) * (a.k + 1) + j] = j < n_acc ? d : j == n_acc ? token : -1;
    }
    if (tid == 0) {
      a.n_acc[b] = n_acc;
      if (a.keep) {
        const int row = a.seq_rows ? a.seq_rows[b] : b;
        a.keep[b] = row >= 0 && row < a.num_rows ? a.lens[row] - a.k + n_acc : 0;
      }
    }
  };
  if (!(rate > 0.0)) {  // a temperature without an answer (the whole workgroup's)
    answer(0, -1);
    return;
  }
  const int per = cdiv(a.chunks, kThreads), c0 = min(tid * per, a.chunks),
            c1 = min(c0 + per, a.chunks);
  const RestSums* rest = a.rest + static_cast<size_t>(b) * a.chunks;
  SamplePick p{0.0, 0.0f, 0.0f, 0, -1};
  const float* maxes = a.maxes + static_cast<size_t>(b) * a.chunks;
  const double* sums = a.sums + static_cast<size_t>(b) * a.chunks;
  if (a.k > 0) {
    p = a.picks[b];
  } else {
    // the only row's maximum
    float m = -INFINITY;
    for (int c = c0; c < c1; ++c) m = max_nan(m, maxes[c]);
    m = wave_max(m);
    if ((tid & 63) == 0) sm_max[w] = m;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kWaves; ++q) m = max_nan(m, sm_max[q]);
    p.mp = m;
  }
  bool both = a.draft && p.n_acc < a.k;
  const double mp = center(p.mp), mq = center(p.mq);
  const E* tr = logits_row<E>(a, b, p.n_acc);
  const E* dr = both ? logits_row<E>(a, b, a.k + 1 + p.n_acc) : tr;

  // L of the two rows' 64-bit sums; no number, 0 or infinite where a row has no distribution
  double lam = 0.0;
  bool sound = true;
  if (both) {
    double se = 0.0, sg = 0.0;
    for (int c = c0; c < c1; ++c) {
      se += rest[c].e;
      sg += rest[c].g;
    }
    se = block_sum(se, sm, tid);
    lam = se / block_sum(sg, sm, tid);
    sound = lam > 0.0 && lam < INFINITY;
  }
  // r (times sum(e)) of this thread's ids of chunk c, and their sum
  const auto ids_of = [&](int c, int v) { return c * kChunk + (tid * NV + v) * N; };
  const auto weights_of = [&](int c, double (&r)[NV][N]) {
    // both products rounded, so that equal probabilities leave exactly nothing
#pragma clang fp contract(off)
    float x[NV][N], y[NV][N];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      load_logits<E>(tr, ids_of(c, v), a.V, x[v]);
      if (both) load_logits<E>(dr, ids_of(c, v), a.V, y[v]);
    }
    double mine = 0.0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int id = ids_of(c, v) + e;
        double t = weight(x[v][e], mp, rate);
        if (both) {
          t = t - lam * weight(y[v][e], mq, rate);
          if (t < 0.0) t = 0.0;  // (a NaN stays)
        } else if (id == p.skip) {
          t = 0.0;
        }
        r[v][e] = id < a.V ? t : 0.0;
        mine += r[v][e];
      }
    }
    return mine;
  };
  // The sums of r over this thread's chunks; plain: of p itself, where p - q, or p without
  // the draft, leaves nothing.
  const auto sum_of = [&](bool plain) {
    double t = 0.0;
    for (int c = c0; c < c1; ++c) {
      if (a.k == 0) t += chunk_sum(sums[c], maxes[c], mp, rate);
      else if (plain) t += rest[c].e;
      else if (!both) t += rest[c].over;
      else if (!rest[c].marked(lam))
        t += fmax(rest[c].over - (lam - p.lam) * rest[c].gp, 0.0) +
             (rest[c].in(lam) ? rest[c].eu - lam * rest[c].gu : 0.0);
    }
    return t;
  };
  double mine = sum_of(false);
  if (both && sound) {
    // marked chunks, in any order: each is one thread's to add
    for (int g = 0; g < per; ++g) {
      const uint64_t m = __ballot(c0 + g < c1 && rest[c0 + g].marked(lam));
      if ((tid & 63) == 0) sm_marked[w] = m;
      __syncthreads();
      for (int q = 0; q < kWaves; ++q) {
        for (uint64_t left = sm_marked[q]; left; left &= left - 1) {
          const int owner = q * 64 + __builtin_ctzll(left);
          double r[NV][N];
          const double s = block_sum(weights_of(owner * per + g, r), sm, tid);
          if (tid == owner) mine += s;
        }
      }
      __syncthreads();
    }
  }
  double R, before = block_prefix(mine, sm, tid, R);
  if (R == 0.0 && (both || p.skip >= 0)) {
    both = false;
    p.skip = -1;
    mine = sum_of(true);
    before = block_prefix(mine, sm, tid, R);
  }
  int32_t token = -1;
  if (sound && R > 0.0) {
    const double place = u * R;
    // the first thread whose running sum passes the place; the last one of any mass
    // where rounding lets none pass
    if (tid == 0) {
      sm_at = kThreads;
      sm_last = -1;
    }
    __syncthreads();
    {
      const uint64_t some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && before + mine > place);
      if ((tid & 63) == 0) {
        if (some) atomicMax(&sm_last, tid + 63 - __builtin_clzll(some));
        if (past) atomicMin(&sm_at, tid + __builtin_ctzll(past));
      }
    }
    __syncthreads();
    const int owner = sm_at < kThreads ? sm_at : sm_last;
    if (tid == owner) sm_ahead = before;
    __syncthreads();
    if (tid == 0) {
      sm_at = a.V;
      sm_last = -1;
    }
    double ahead = sm_ahead;
    for (int c = owner * per; c < min((owner + 1) * per, a.chunks); ++c) {
      double r[NV][N], all;
      double at = ahead + block_prefix(weights_of(c, r), sm, tid, all);
      ahead += all;
      int first = a.V, last = -1;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          at += r[v][e];
          if (r[v][e] > 0.0) {
            last = ids_of(c, v) + e;
            if (at > place && first == a.V) first = last;
          }
        }
      }
      // (ids grow with the lane)
      const uint64_t some = __ballot(last >= 0), past = __ballot(first < a.V);
      if (some && (tid & 63) == 63 - __builtin_clzll(some)) atomicMax(&sm_last, last);
      if (past && (tid & 63) == __builtin_ctzll(past)) atomicMin(&sm_at, first);
      __syncthreads();
      if (sm_at < a.V) break;
    }
    token = sm_at < a.V ? sm_at : sm_last;
  }
  answer(p.n_acc, token);
}

// Workgroups of the stats launch: 8 per compute unit, what the chip holds at once in bf16
// (58 and 63 registers). In fp32 (84 and 90) it holds 5, and the others follow.
constexpr int kStatGrid = 2048;

struct SampleCfg {
  int rows, chunks;
  size_t sums, maxes, rest, picks, bytes;  // offsets of the workspace's parts
};

static SampleCfg sample_cfg(int B, int k, int V, bool draft) {
  SampleCfg c{};
  c.rows = draft ? 2 * k + 1 : k + 1;
  c.chunks = cdiv(V, kChunk);
  const size_t parts = static_cast<size_t>(B) * c.rows * c.chunks;
  size_t at = 0;
  const auto take = [&](size_t n) {
    const size_t was = at;
    at += (n + 15) & ~static_cast<size_t>(15);
    return was;
  };
  c.sums = take(parts * sizeof(double));
  c.maxes = take(parts * sizeof(float));
  c.rest = take(k ? static_cast<size_t>(B) * c.chunks * sizeof(RestSums) : 0);
  c.picks = take(static_cast<size_t>(B) * sizeof(SamplePick));
  c.bytes = at;
  return c;
}

template <typename E>
static void launch_sample(const SampleArgs& a, hipStream_t st) {
  const dim3 stats(std::min(kStatGrid, cdiv(a.B * a.rows * a.chunks, kWaves))), wg(kThreads);
  if (a.k > 0) {
    hipLaunchKernelGGL((sample_stats_kernel<E, false>), stats, wg, 0, st, a);
    hipLaunchKernelGGL(sample_rest_kernel<E>, dim3(a.B * cdiv(a.chunks, kWaves)), wg,
                       static_cast<size_t>(a.rows) * (sizeof(double) + sizeof(float)), st, a);
  } else {
    hipLaunchKernelGGL((sample_stats_kernel<E, true>), stats, wg, 0, st, a);
  }
  hipLaunchKernelGGL(sample_pick_kernel<E>, dim3(a.B), wg, 0, st, a);
}

}  // namespace kve

using namespace kve;

// Drafts a sequence may have: a thread each in decide().
constexpr int kSampleMaxDrafts = kThreads;

extern "C" size_t kve_sample_workspace_bytes(int num_seqs, int k, int vocab, int dtype) {
  if (num_seqs <= 0 || k < 0 || k > kSampleMaxDrafts || vocab <= 0 ||
      (dtype != KVE_DTYPE_BF16 && dtype != KVE_DTYPE_F32))
    return 0;
  return std::max(sample_cfg(num_seqs, k, vocab, true).bytes,
                  sample_cfg(num_seqs, k, vocab, false).bytes);
}

extern "C" int kve_sample_verify(const void* target, int64_t target_seq_stride,
                                 int64_t target_pos_stride, const void* draft,
                                 int64_t draft_seq_stride, int64_t draft_pos_stride,
                                 const int32_t* drafts, const float* u_accept,
                                 const float* u_sample, const float* temperatures,
                                 double temperature, const int32_t* lens, int num_rows,
                                 const int32_t* seq_rows, int num_seqs, int k, int vocab,
                                 int dtype, int32_t* n_acc, int32_t* emitted, int32_t* keep_lens,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (num_seqs == 0) return KVE_OK;
  KVE_REQUIRE(target && u_sample && n_acc && emitted && (k == 0 || (drafts && u_accept)),
              "kve_sample_verify: null pointer argument");
  KVE_REQUIRE(num_seqs > 0 && k >= 0 && k <= kSampleMaxDrafts && vocab > 0 && vocab <= (1 << 30),
              "kve_sample_verify: %d sequences, k = %d (at most %d), vocabulary %d", num_seqs, k,
              kSampleMaxDrafts, vocab);
  KVE_REQUIRE(dtype == KVE_DTYPE_BF16 || dtype == KVE_DTYPE_F32, "kve_sample_verify: dtype %d",
              dtype);
  // (the range of positive 32-bit numbers, over which no exponent leaves 64 bits)
  KVE_REQUIRE(temperatures || (temperature > 0x1p-150 && temperature < 0x1.ffffffp127),
              "kve_sample_verify: temperature %g", temperature);
  KVE_REQUIRE(!keep_lens || (lens && num_rows > 0), "kve_sample_verify: keep_lens needs lens");
  const size_t esz = dtype == KVE_DTYPE_BF16 ? 2 : 4;
  KVE_REQUIRE(((reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft)) &
               (esz - 1)) == 0,
              "kve_sample_verify: logits are not aligned to their type");
  const SampleCfg c = sample_cfg(num_seqs, k, vocab, draft != nullptr && k > 0);
  KVE_REQUIRE(static_cast<long long>(num_seqs) * c.rows * c.chunks < (1ll << 30),
              "kve_sample_verify: %d x %d rows of %d too large for one launch", num_seqs, c.rows,
              vocab);
  KVE_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              "kve_sample_verify: workspace required (16-byte aligned)");
  if (workspace_bytes < c.bytes) {
    set_error("kve_sample_verify: workspace %zu bytes, need %zu", workspace_bytes, c.bytes);
    return KVE_EWORKSPACE;
  }
  char* ws = static_cast<char*>(workspace);
  SampleArgs a{};
  a.target = target;
  a.draft = k > 0 ? draft : nullptr;
  a.ts = target_seq_stride;
  a.tp = target_pos_stride;
  a.ds = draft_seq_stride;
  a.dp = draft_pos_stride;
  a.drafts = drafts;
  a.u_accept = u_accept;
  a.u_sample = u_sample;
  a.temps = temperatures;
  a.temp = temperature;
  a.lens = lens;
  a.seq_rows = seq_rows;
  a.num_rows = num_rows;
  a.B = num_seqs;
  a.k = k;
  a.V = vocab;
  a.rows = c.rows;
  a.chunks = c.chunks;
  a.n_acc = n_acc;
  a.emitted = emitted;
  a.keep = keep_lens;
  a.sums = reinterpret_cast<double*>(ws + c.sums);
  a.maxes = reinterpret_cast<float*>(ws + c.maxes);
  a.rest = reinterpret_cast<RestSums*>(ws + c.rest);
  a.picks = reinterpret_cast<SamplePick*>(ws + c.picks);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == KVE_DTYPE_BF16) launch_sample<uint16_t>(a, st);
  else launch_sample<float>(a, st);
  return check_launch("kve_sample_verify");
}
