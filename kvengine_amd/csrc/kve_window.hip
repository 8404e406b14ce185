// Attention over the paged cache with a sliding window and sinks, and over a cache held
// in 8 bits (kve_paged_window_attn, kve_paged_q8_attn). The counterpart in the reference
// is its gather and masked SDPA (kvengine/paged.py:315-331, forward.py:85-144), which knows
// neither a window (it refuses such models) nor a quantised cache.
//
// The mathematics. The query at position p sees key j where j <= p and (j > p - window or
// j < sinks): softmax(q k^T * scale) v over those, one pass with the running maximum m and
// sum l of the softmax. In an 8-bit cache k = c s_k and v = c s_v with one scale per block
// and head: s_k multiplies the scores, s_v the probabilities, and the products are taken
// with the codes.
//
// Work. Rows: the G = Hq / Hkv query heads of a kv head times the new tokens (row r =
// t G + head). A wave holds MT tiles of 16 rows and walks the keys they see in steps of
// SK = 16 NT keys (NT = 4 / bytes of an element: 16 fp32, 32 bf16, 64 8-bit): first the steps
// that hold sinks, then those of the window; what lies between is not read. A workgroup is
// four waves, RW row waves times KW = 4 / RW key waves that take steps in turn and are folded
// through LDS; a long walk is cut into chunks of steps, a workgroup each, that a second launch
// joins in chunk order.
//
// A step. Every lane loads 16 bytes at a time straight into registers: of K, lane (lr, lg)
// of score product t reads key 4 NT (lr / 4) + 4 t + lr % 4 of the step, of V channel
// 16 dt + lr, keys 4 NT lg ... Scores are S^T = K Q^T (16x16 matrix products, rows of K on
// the M side): lane (lr, lg) then holds the scores of row lr and keys 4 NT lg + 4 t + i,
// which are the keys of its V bytes, so P^T goes back as an operand of O^T = V^T P^T without
// leaving the lane. K and V are read by the one wave that needs them (other row waves' reads
// hit the caches), so nothing is staged and no barrier stands in the walk: while one step's
// probabilities are taken the next one's K is on its way, and its V during the scores.
//
// Numbers. bf16: products in bf16, P as the sum of two bf16 (16 bits of it). fp32: fp32
// products. 8 bits: codes are exact in fp16, so the products are fp16's: q is scaled to the
// fp16 range by a power of two per row (exact for bf16; fp32 as the sum of two fp16, 22
// bits), P s_v by one per walk (11 bits of it for bf16 queries, 22 for fp32). Sums, m and l
// are fp32.
//
// Values that a row must not see. A masked score is replaced, not added to, so that nothing
// of its key remains. In V a masked infinity or NaN would be 0 * inf: steps that some
// row sees in part are taken without the non-finite values, which are then added to the rows
// that do see them (add_nonfinite). Other steps are seen whole by every row.

#include "kve_q8.h"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace kve {

enum class Pool { kBf16, kF32, kInt8, kE4m3 };

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct WindowArgs {
  const void* q;
  const uint8_t *k, *v;
  const float *ks, *vs;  // [num_blocks][Hkv], 8-bit pools
  void* out;
  const int32_t *tables, *seq_rows, *start_pos, *q_lens;
  float* part_o;   // [B][Hkv][splits][rows][D]
  float* part_ml;  // [B][Hkv][splits][rows][2]
  int B, Tq, Hq, Hkv, G, bs, tpb, max_blocks, num_rows, num_blocks, max_ctx;
  int window, sinks;
  int rw, row_groups, chunk, splits;  // chunk: steps of a workgroup
  float scale_log2;
  uint32_t g_magic, tpb_magic;
};

constexpr int kWinThreads = 256;
constexpr float kNone = -1.0e30f;  // the maximum of a row that has seen no key

// n / d for 0 <= n < 2^16 with magic = ceil(2^32 / d), d >= 2 (the host checks the range)
__device__ __forceinline__ int div_magic(int n, int d, uint32_t magic) {
  return d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), magic));
}

struct WinSeq {
  int row, start, T;  // T = 0: nothing to do
};

__device__ __forceinline__ WinSeq win_seq(const WindowArgs& a, int b) {
  WinSeq s{0, 0, 0};
  const int row = a.seq_rows ? a.seq_rows[b] : b;
  if (row < 0 || row >= a.num_rows) return s;
  const int start = a.start_pos[row];
  const int T = a.q_lens ? min(a.q_lens[b], a.Tq) : a.Tq;
  if (T <= 0 || start < 0 || start > a.max_ctx - T) return s;
  return WinSeq{row, start, T};
}

// The steps of SK keys that the rows [row0, row1) see: steps 0 .. sinks - 1, then
// first .. first + rest - 1.
struct Walk {
  int p0, p1;  // positions of the first and the last query
  int sinks, first, total;
  __device__ __forceinline__ int step(int i) const { return i < sinks ? i : first + i - sinks; }
};

template <int SK>
__device__ __forceinline__ Walk walk_of(const WindowArgs& a, const WinSeq& s, int row0, int row1) {
  Walk w;
  w.p0 = s.start + div_magic(row0, a.G, a.g_magic);
  w.p1 = s.start + div_magic(row1 - 1, a.G, a.g_magic);
  w.first = w.p0 >= a.window ? (w.p0 - a.window + 1) / SK : 0;
  w.sinks = min((a.sinks + SK - 1) / SK, w.first);
  w.total = w.sinks + w.p1 / SK - w.first + 1;
  return w;
}

// ---- element types ----------------------------------------------------------------

template <Pool P>
struct PoolOf {
  static constexpr int ES = P == Pool::kF32 ? 4 : P == Pool::kBf16 ? 2 : 1;
  static constexpr int NT = 4 / ES;    // 16-key tiles of a step
  static constexpr int SK = 16 * NT;
  static constexpr bool Q8B = ES == 1;
};

// 4 codes -> 4 fp16, exact: int8 + 128 set into the low bits of 1024 + x, less 1152.
template <Pool P>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (P == Pool::kInt8) {
    w ^= 0x80808080u;
    const f16x2 off = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off);
  } else {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  }
}

// 16 codes -> the two 8-value operands they make
template <Pool P>
__device__ __forceinline__ void codes_to_frags(u32x4 c, u32x4 (&f)[2]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t lo, hi;
    codes_to_f16<P>(c[w], lo, hi);
    f[w >> 1][2 * (w & 1)] = lo;
    f[w >> 1][2 * (w & 1) + 1] = hi;
  }
}

__device__ __forceinline__ f32x4 mfma16x16x32_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two floats -> packed fp16 pair, to nearest even
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
}

// The pair and what it leaves of a and b
__device__ __forceinline__ uint32_t split_f16x2(float& a, float& b) {
  const uint32_t h = pack_f16x2(a, b);
  const f16x2 v = __builtin_bit_cast(f16x2, h);
  a -= static_cast<float>(v[0]);
  b -= static_cast<float>(v[1]);
  return h;
}
__device__ __forceinline__ uint32_t split_bf16x2(float& a, float& b) {
  const uint32_t h = pack_bf16x2(a, b);
  a -= __uint_as_float(h << 16);
  b -= __uint_as_float(h & 0xffff0000u);
  return h;
}

// The non-finite values of 16 bytes set to 0; whether there were any.
template <Pool P>
__device__ __forceinline__ bool drop_nonfinite(u32x4& x) {
  uint32_t any = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (P == Pool::kBf16) {
      const uint32_t f = ((x[w] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
      x[w] &= ~((f >> 15) * 0xffffu);
      any |= f;
    } else if constexpr (P == Pool::kF32) {
      const bool f = (x[w] & 0x7f800000u) == 0x7f800000u;
      x[w] = f ? 0u : x[w];
      any |= f;
    } else if constexpr (P == Pool::kE4m3) {
      const uint32_t f = ((x[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
      x[w] &= ~((f >> 7) * 0xffu);
      any |= f;
    }
  }
  return any != 0;
}

// A V value if it is not finite, else 0.
template <Pool P>
__device__ __forceinline__ float nonfinite_of(const uint8_t* p) {
  float v = 0.0f;
  if constexpr (P == Pool::kBf16) v = bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
  if constexpr (P == Pool::kF32) v = *reinterpret_cast<const float*>(p);
  if constexpr (P == Pool::kE4m3) return (*p & 0x7f) == 0x7f ? NAN : 0.0f;
  return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? v : 0.0f;
}

// ---- the walk ---------------------------------------------------------------------
// PARTS: 16-bit parts that P is taken as (and, over 8-bit pools, q): 8-bit pools 1 for bf16
// queries and 2 for fp32 ones, bf16 2; fp32 takes P whole (1).
template <Pool P, int PARTS, int D, int MT>
__global__ __launch_bounds__(kWinThreads, 2) void window_attn_kernel(WindowArgs a) {
  using X = PoolOf<P>;
  constexpr int ES = X::ES, NT = X::NT, SK = X::SK;
  constexpr bool Q8B = X::Q8B, F32 = P == Pool::kF32;
  constexpr bool QBF = P == Pool::kBf16 || (Q8B && PARTS == 1);  // q and out in bf16
  constexpr int QP = Q8B ? PARTS : 1;
  constexpr int NJ = D * ES / 64;  // 16-byte pieces of a K row per lane
  constexpr int DT = D / 16;
  constexpr int NF = F32 ? D / 16 : D / 32;  // q fragments of 16 bytes
  constexpr int BATCH = 64 / NT;             // steps whose block ids a wave holds
  extern __shared__ float sm[];

  const int tid = threadIdx.x, l = tid & 63, lr = l & 15, lg = l >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  int u = blockIdx.x;
  const int rg = u % a.row_groups;
  u /= a.row_groups;
  const int c = u % a.splits;
  u /= a.splits;
  const int kvh = u % a.Hkv, b = u / a.Hkv;
  const int KW = 4 / a.rw, rwi = wid / KW, kw = wid - rwi * KW;
  const WinSeq s = win_seq(a, b);
  const int R = a.G * s.T, rows = 16 * MT * a.rw;
  if (rg * rows >= R) return;
  const int row0 = rg * rows + rwi * 16 * MT, row1 = min(R, row0 + 16 * MT);
  const bool active = row0 < R;
  const Walk w = walk_of<SK>(a, s, active ? row0 : 0, active ? row1 : 1);
  const int chunks = active ? cdiv(w.total, a.chunk) : 0;
  // (row waves of one workgroup may end at different chunks; they meet at the fold only)
  const int end = c < chunks ? min(w.total, (c + 1) * a.chunk) : 0;

  f32x4 acc[MT][DT];
  float m[MT], lsum[MT];
  int qpos[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = f32x4{0, 0, 0, 0};
    m[mt] = kNone;
    lsum[mt] = 0.0f;
  }
  float ref = kMinScale;  // acc is in units of it: a power of two that no s_v seen so far exceeds

  if (c * a.chunk + kw < end) {
    // q: the lane's channels of row lr of each tile, in the order of its K pieces
    u32x4 qf[MT][QP][NF];
    float rf[MT];  // score -> exponent of 2
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = min(row0 + mt * 16 + lr, R - 1);
      const int t = div_magic(r, a.G, a.g_magic), h = kvh * a.G + r - t * a.G;
      qpos[mt] = s.start + t;
      const size_t at = ((static_cast<size_t>(b) * a.Tq + t) * a.Hq + h) * D;
      rf[mt] = a.scale_log2;
      if constexpr (!Q8B) {
        const uint8_t* qp = static_cast<const uint8_t*>(a.q) + at * ES + lg * 16;
#pragma unroll
        for (int j = 0; j < NF; ++j) qf[mt][0][j] = *reinterpret_cast<const u32x4*>(qp + j * 64);
      } else {
        // channels 64 j + 16 lg + 8 f .. of fragment 2 j + f
        float x[NF][8];
        float top = 0.0f;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const size_t ch = at + (f >> 1) * 64 + lg * 16 + (f & 1) * 8;
          if constexpr (QBF) {
            const u32x4 raw = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + ch);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              x[f][e] = __uint_as_float(e & 1 ? raw[e >> 1] & 0xffff0000u : raw[e >> 1] << 16);
          } else {
            const float* qp = static_cast<const float*>(a.q) + ch;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[f][e] = qp[e];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[f][e]));
        }
        top = max_across_groups(top);
        // the row's largest value to [2^13, 2^14): what falls below fp16's steps of 2^-24
        // there is below 2^-38 of it
        int ex = 0;
        if (top > 0.0f && top < INFINITY) frexpf(top, &ex);
        rf[mt] = ldexpf(a.scale_log2, ex - 14);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[f][e] = ldexpf(x[f][e], 14 - ex);
#pragma unroll
          for (int p = 0; p < QP; ++p) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              qf[mt][p][f][e] = p + 1 < QP ? split_f16x2(x[f][2 * e], x[f][2 * e + 1])
                                           : pack_f16x2(x[f][2 * e], x[f][2 * e + 1]);
          }
        }
      }
    }

    const int32_t* table = a.tables + static_cast<size_t>(s.row) * a.max_blocks;
    const int last_tile = w.p1 >> 4;
    // the lane's K row and V keys within a step
    const int kk = 4 * NT * (lr >> 2) + (lr & 3), vk = 4 * NT * lg;
    const int ktile = kk >> 4, vtile = vk >> 4;
    const size_t kin = static_cast<size_t>(kk & 15) * D * ES + lg * 16;
    const size_t vrow = static_cast<size_t>(a.bs) * ES;
    const size_t vin = lr * vrow + (vk & 15) * ES;
    const size_t tile_bytes = static_cast<size_t>(a.bs) * D * ES;  // a (block, head)

    u32x4 kf[NT * NJ], vf[DT];
    int ids = 0;              // of the batch: tile lane's (block * Hkv + kvh) * tpb + part of it
    float ksl = 0, vsl = 0;   // its scales
    const auto tile_at = [&](int i, int tile) {  // (block, head) and the tile's place in it
      const int id = __shfl(ids, i * NT + tile);
      return id;
    };
    const auto load_k = [&](int i) {
      const int id = tile_at(i, ktile);
      const int bh = a.tpb == 1 ? id : id / a.tpb, part = a.tpb == 1 ? 0 : id - bh * a.tpb;
      const uint8_t* p = a.k + static_cast<size_t>(bh) * tile_bytes +
                         static_cast<size_t>(part) * 16 * D * ES + kin;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          kf[t * NJ + j] = *reinterpret_cast<const u32x4*>(p + t * 4 * D * ES + j * 64);
      }
    };
    const auto load_v = [&](int i) {
      const int id = tile_at(i, vtile);
      const int bh = a.tpb == 1 ? id : id / a.tpb, part = a.tpb == 1 ? 0 : id - bh * a.tpb;
      const uint8_t* p = a.v + static_cast<size_t>(bh) * tile_bytes +
                         static_cast<size_t>(part) * 16 * ES + vin;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        vf[dt] = *reinterpret_cast<const u32x4*>(p + dt * 16 * vrow);
    };

    for (int i0 = c * a.chunk + kw; i0 < end; i0 += BATCH * KW) {
      const int steps = min(BATCH, cdiv(end - i0, KW));
      {
        // lane: tile l % NT of the batch's step l / NT (past the last: it again)
        const int st = w.step(i0 + min(l / NT, steps - 1) * KW);
        const int tile = min(st * NT + l % NT, last_tile);
        const int lb = a.tpb == 1 ? tile : tile / a.tpb;
        const int blk = table[lb];  // within the table: start + T <= max_ctx <= its blocks
        const int bh = (static_cast<unsigned>(blk) < static_cast<unsigned>(a.num_blocks) ? blk : 0) * a.Hkv + kvh;
        ids = bh * a.tpb + tile - lb * a.tpb;
        if constexpr (Q8B) {
          ksl = a.ks[bh];
          vsl = a.vs[bh];
          const int k0 = tile * 16;
          const bool seen = k0 + 15 > w.p0 - a.window || k0 < a.sinks;
          float top = seen && vsl < INFINITY ? vsl : 0.0f;
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
          top = max_across_groups(top);
          if (top > ref) {  // (the same in every lane)
            int ex;
            frexpf(top, &ex);
            const float to = ldexpf(1.0f, min(ex, 127)), f = ref / to;
            ref = to;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= f;
            }
          }
        }
      }
      load_k(0);
      load_v(0);
      for (int i = 0; i < steps; ++i) {
        const int k0 = w.step(i0 + i * KW) * SK;
        f32x4 sc[MT][NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) sc[mt][t] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            if constexpr (F32) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
                  sc[mt][t] = mfma16x16x4_f32(__uint_as_float(kf[t * NJ + j][e]),
                                              __uint_as_float(qf[mt][0][j][e]), sc[mt][t]);
              }
            } else if constexpr (Q8B) {
              u32x4 f[2];
              codes_to_frags<P>(kf[t * NJ + j], f);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                  for (int p = 0; p < QP; ++p)
                    sc[mt][t] = mfma16x16x32_f16(f[e], qf[mt][p][2 * j + e], sc[mt][t]);
                }
              }
            } else {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
                sc[mt][t] = mfma16x16x32_bf16(kf[t * NJ + j], qf[mt][0][j], sc[mt][t]);
            }
          }
        }
        const bool more = i + 1 < steps;
        if (more) load_k(i + 1);
        float ks = 1.0f, vs = 1.0f;
        if constexpr (Q8B) {
          ks = __shfl(ksl, i * NT + lg);
          vs = __shfl(vsl, i * NT + lg) * (0x1p14f / ref);
        }
        // seen whole by every row of the wave
        const bool whole = k0 + SK - 1 <= w.p0 && (k0 > w.p1 - a.window || k0 + SK <= a.sinks);
        bool dropped = false;
        if (!whole && P != Pool::kInt8) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) dropped |= drop_nonfinite<P>(vf[dt]);
        }
        u32x4 pf[MT][PARTS][F32 ? 1 : NT / 2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float f = Q8B ? rf[mt] * ks : rf[mt];
          float x[4 * NT];
          float top = kNone;
#pragma unroll
          for (int n = 0; n < 4 * NT; ++n) x[n] = sc[mt][n >> 2][n & 3] * f;
          if (!whole) {
#pragma unroll
            for (int n = 0; n < 4 * NT; ++n) {
              const int key = k0 + 4 * NT * lg + n;
              const bool sees = key <= qpos[mt] && (key > qpos[mt] - a.window || key < a.sinks);
              x[n] = sees ? x[n] : -INFINITY;
            }
          }
#pragma unroll
          for (int n = 0; n < 4 * NT; ++n) top = fmaxf(top, x[n]);
          top = max_across_groups(top);
          if (__any(top > m[mt])) {
            const float to = fmaxf(m[mt], top), al = __builtin_amdgcn_exp2f(m[mt] - to);
            m[mt] = to;
            lsum[mt] *= al;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= al;
          }
          float add = 0.0f;
#pragma unroll
          for (int n = 0; n < 4 * NT; ++n) {
            x[n] = __builtin_amdgcn_exp2f(x[n] - m[mt]);
            add += x[n];
            // (0 * s_v of a block whose scale is no number stays 0)
            if constexpr (Q8B) x[n] = whole || x[n] > 0.0f || x[n] != x[n] ? x[n] * vs : 0.0f;
          }
          lsum[mt] += add;
          if constexpr (F32) {
#pragma unroll
            for (int n = 0; n < 4; ++n) pf[mt][0][0][n] = __float_as_uint(x[n]);
          } else {
#pragma unroll
            for (int n = 0; n < 2 * NT; ++n) {
#pragma unroll
              for (int p = 0; p < PARTS; ++p) {
                uint32_t h;
                if constexpr (Q8B)
                  h = p + 1 < PARTS ? split_f16x2(x[2 * n], x[2 * n + 1]) : pack_f16x2(x[2 * n], x[2 * n + 1]);
                else
                  h = p + 1 < PARTS ? split_bf16x2(x[2 * n], x[2 * n + 1]) : pack_bf16x2(x[2 * n], x[2 * n + 1]);
                pf[mt][p][n >> 2][n & 3] = h;
              }
            }
          }
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
                acc[mt][dt] = mfma16x16x4_f32(__uint_as_float(vf[dt][e]),
                                              __uint_as_float(pf[mt][0][0][e]), acc[mt][dt]);
            }
          } else if constexpr (Q8B) {
            u32x4 f[2];
            codes_to_frags<P>(vf[dt], f);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
                  acc[mt][dt] = mfma16x16x32_f16(f[e], pf[mt][p][e], acc[mt][dt]);
              }
            }
          } else {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
              for (int p = 0; p < PARTS; ++p)
                acc[mt][dt] = mfma16x16x32_bf16(vf[dt], pf[mt][p][0], acc[mt][dt]);
            }
          }
        }
        if (__any(dropped)) {
          // rare: the step's keys one by one, their non-finite values to the rows that see them
#pragma unroll 1
          for (int n = 0; n < SK; ++n) {
            const int key = k0 + n;
            if (key > w.p1) break;
            const int id = __shfl(ids, i * NT + (n >> 4));
            const int bh = id / a.tpb, part = id - bh * a.tpb;
            const uint8_t* p = a.v + static_cast<size_t>(bh) * tile_bytes +
                               static_cast<size_t>(4 * lg) * vrow + (part * 16 + (n & 15)) * ES;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float v = nonfinite_of<P>(p + (dt * 16 + e) * vrow);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  const bool sees = key <= qpos[mt] && (key > qpos[mt] - a.window || key < a.sinks);
                  acc[mt][dt][e] += sees ? v : 0.0f;
                }
              }
            }
          }
        }
        if (more) load_v(i + 1);
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      lsum[mt] = sum_across_groups(lsum[mt]);
      if constexpr (Q8B) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= ref * 0x1p-14f;
      }
    }
  }

  // the key waves of a row wave, in order, into its first
  if (KW > 1) {
    constexpr int WAVE = MT * (DT * 256 + 32);  // floats a wave leaves
    float* mine = sm + static_cast<size_t>(rwi * (KW - 1) + kw - 1) * WAVE;
    if (kw > 0) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (lg == 0) {
          mine[MT * DT * 256 + mt * 32 + 2 * lr] = m[mt];
          mine[MT * DT * 256 + mt * 32 + 2 * lr + 1] = lsum[mt];
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          *reinterpret_cast<f32x4*>(mine + ((mt * DT + dt) * 64 + l) * 4) = acc[mt][dt];
      }
    }
    __syncthreads();
    if (kw > 0) return;
    for (int o = 0; o < KW - 1; ++o) {
      const float* other = sm + static_cast<size_t>(rwi * (KW - 1) + o) * WAVE;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float mo = other[MT * DT * 256 + mt * 32 + 2 * lr];
        const float lo = other[MT * DT * 256 + mt * 32 + 2 * lr + 1];
        const float to = fmaxf(m[mt], mo);
        const float al = __builtin_amdgcn_exp2f(m[mt] - to), be = __builtin_amdgcn_exp2f(mo - to);
        m[mt] = to;
        lsum[mt] = lsum[mt] * al + lo * be;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          acc[mt][dt] = acc[mt][dt] * al +
                        *reinterpret_cast<const f32x4*>(other + ((mt * DT + dt) * 64 + l) * 4) * be;
      }
    }
  }
  if (c >= chunks) return;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = row0 + mt * 16 + lr;
    if (r >= R) continue;
    if (chunks == 1) {
      const int t = div_magic(r, a.G, a.g_magic), h = kvh * a.G + r - t * a.G;
      const size_t at = ((static_cast<size_t>(b) * a.Tq + t) * a.Hq + h) * D + 4 * lg;
      const float inv = 1.0f / lsum[mt];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f32x4 y = acc[mt][dt] * inv;
        if constexpr (QBF)
          *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + at + dt * 16) =
              u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        else
          *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at + dt * 16) = y;
      }
    } else {
      const size_t slot =
          ((static_cast<size_t>(b) * a.Hkv + kvh) * a.splits + c) * a.row_groups * rows + r;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<f32x4*>(a.part_o + slot * D + dt * 16 + 4 * lg) = acc[mt][dt];
      if (lg == 0) {
        a.part_ml[slot * 2] = m[mt];
        a.part_ml[slot * 2 + 1] = lsum[mt];
      }
    }
  }
}

// Rows whose walk has several chunks: the chunks' states joined in chunk order, a wave
// per row, lane l channels l, l + 64.
template <int SK, int D, bool OUT_BF16>
__global__ __launch_bounds__(kWinThreads) void window_merge_kernel(WindowArgs a, int wave_rows) {
  const int l = threadIdx.x & 63;
  const int rmax = a.G * a.Tq;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * (kWinThreads / 64) + (threadIdx.x >> 6);
  if (u >= static_cast<int64_t>(a.B) * a.Hkv * rmax) return;
  const int r = static_cast<int>(u % rmax), bh = static_cast<int>(u / rmax);
  const int b = bh / a.Hkv, kvh = bh - b * a.Hkv;
  const WinSeq s = win_seq(a, b);
  const int R = a.G * s.T;
  if (r >= R) return;
  const int row0 = r / wave_rows * wave_rows;
  const Walk w = walk_of<SK>(a, s, row0, min(R, row0 + wave_rows));
  const int chunks = cdiv(w.total, a.chunk);
  if (chunks == 1) return;
  const size_t per = static_cast<size_t>(a.row_groups) * wave_rows * a.rw;
  const size_t slot0 = static_cast<size_t>(bh) * a.splits * per + r;
  constexpr int N = D / 64;
  float m = kNone, sum = 0.0f, o[N];
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = 0.0f;
  for (int c = 0; c < chunks; ++c) {
    const size_t slot = slot0 + c * per;
    const float mc = a.part_ml[slot * 2], lc = a.part_ml[slot * 2 + 1];
    const float to = fmaxf(m, mc), al = __builtin_amdgcn_exp2f(m - to), be = __builtin_amdgcn_exp2f(mc - to);
    m = to;
    sum = sum * al + lc * be;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = o[e] * al + a.part_o[slot * D + e * 64 + l] * be;
  }
  const int t = div_magic(r, a.G, a.g_magic), h = kvh * a.G + r - t * a.G;
  const size_t at = ((static_cast<size_t>(b) * a.Tq + t) * a.Hq + h) * D + l;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = o[e] / sum;
    if constexpr (OUT_BF16) static_cast<uint16_t*>(a.out)[at + e * 64] = f32_to_bf16(y);
    else static_cast<float*>(a.out)[at + e * 64] = y;
  }
}

// ---- launch -------------------------------------------------------------------------

// Workgroups that a launch should have before walks are cut: two per compute unit.
constexpr int kFill = 512;
// Steps of a key wave below which a walk is not cut further.
constexpr int kMinSteps = 2;

struct WindowCfg {
  int mt, rw, row_groups, chunk, splits;
  size_t ml, bytes;  // offset of part_ml, the workspace's size
};

// sk: keys of a step
static WindowCfg window_cfg(int B, int Tq, int Hq, int Hkv, int D, int max_ctx, int window,
                            int sinks, int sk) {
  WindowCfg c{};
  const int R = Hq / Hkv * Tq;
  const int most = D == 64 ? 4 : 2;  // tiles whose state stays in a wave's registers
  c.mt = R <= 16 ? 1 : R <= 32 ? 2 : most;
  c.rw = R <= 16 * c.mt ? 1 : R <= 32 * c.mt ? 2 : 4;
  c.row_groups = cdiv(R, 16 * c.mt * c.rw);
  const int kw = 4 / c.rw;
  // the longest walk: the window of a wave's first query to its last
  const int64_t keys = std::min<int64_t>(
      max_ctx, static_cast<int64_t>(window) + cdiv(16 * c.mt, Hq / Hkv) + 1);
  int64_t steps = keys / sk + 2;
  if (keys < max_ctx) steps += cdiv(std::min(sinks, max_ctx), sk);
  const int64_t units = static_cast<int64_t>(B) * Hkv * c.row_groups;
  const int64_t want = std::max<int64_t>(1, kFill / units);
  int64_t chunk = std::max<int64_t>((steps + want - 1) / want, kMinSteps * kw);
  chunk = (chunk + kw - 1) / kw * kw;
  c.splits = static_cast<int>((steps + chunk - 1) / chunk);
  c.chunk = static_cast<int>(chunk);
  if (c.splits > 1) {
    const size_t slots = static_cast<size_t>(B) * Hkv * c.splits * c.row_groups * 16 * c.mt * c.rw;
    c.ml = slots * D * sizeof(float);
    c.bytes = c.ml + slots * 2 * sizeof(float);
  }
  return c;
}

template <Pool P, int PARTS, int D, int MT>
static int launch_walk(const WindowArgs& a, int64_t grid, hipStream_t st) {
  const auto kernel = window_attn_kernel<P, PARTS, D, MT>;
  const int kw = 4 / a.rw;
  const size_t lds = static_cast<size_t>(a.rw) * (kw - 1) * MT * (D * 16 + 32) * sizeof(float);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kWinThreads), lds, st, a);
  return KVE_OK;
}

template <Pool P, int PARTS, int D>
static int launch_window(const WindowArgs& a, const WindowCfg& c, hipStream_t st) {
  const int64_t grid = static_cast<int64_t>(a.B) * a.Hkv * c.splits * c.row_groups;
  int rc = KVE_OK;
  if (c.mt == 1) rc = launch_walk<P, PARTS, D, 1>(a, grid, st);
  else if (c.mt == 2) rc = launch_walk<P, PARTS, D, 2>(a, grid, st);
  else if constexpr (D == 64) rc = launch_walk<P, PARTS, D, 4>(a, grid, st);
  if (rc) return rc;
  if (c.splits > 1) {
    constexpr bool bf = P == Pool::kBf16 || (PoolOf<P>::Q8B && PARTS == 1);
    const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * a.G * a.Tq;
    hipLaunchKernelGGL((window_merge_kernel<PoolOf<P>::SK, D, bf>),
                       dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(kWinThreads), 0, st, a,
                       16 * c.mt);
  }
  return check_launch("paged window attention");
}

template <Pool P, int PARTS>
static int launch_window_d(const WindowArgs& a, const WindowCfg& c, int D, hipStream_t st) {
  return D == 64 ? launch_window<P, PARTS, 64>(a, c, st) : launch_window<P, PARTS, 128>(a, c, st);
}

static int step_keys(int pool_dtype) {
  return pool_dtype == KVE_DTYPE_F32 ? 16 : pool_dtype == KVE_DTYPE_BF16 ? 32 : 64;
}

static bool window_sizes_ok(int B, int Tq, int Hq, int Hkv, int D, int max_ctx, int window, int sinks) {
  return B > 0 && Tq > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && (D == 64 || D == 128) &&
         max_ctx > 0 && window >= 0 && sinks >= 0 && static_cast<int64_t>(Hq / Hkv) * Tq < 65536;
}

}  // namespace kve

using namespace kve;

extern "C" size_t kve_window_workspace_bytes(int num_seqs, int q_len, int num_q_heads,
                                             int num_kv_heads, int head_dim, int max_ctx,
                                             int window, int sinks, int pool_dtype) {
  if (!window_sizes_ok(num_seqs, q_len, num_q_heads, num_kv_heads, head_dim, max_ctx, window, sinks))
    return 0;
  return window_cfg(num_seqs, q_len, num_q_heads, num_kv_heads, head_dim, max_ctx,
                    window > 0 ? window : INT32_MAX, sinks, step_keys(pool_dtype))
      .bytes;
}

extern "C" int kve_paged_window_attn(const void* q, const void* k_layer, const void* v_layer,
                                     const float* k_scale, const float* v_scale,
                                     const int32_t* block_tables, const int32_t* seq_rows,
                                     const int32_t* start_pos, const int32_t* q_lens, int num_seqs,
                                     int q_len, int num_q_heads, int num_kv_heads, int head_dim,
                                     int block_size, int max_blocks, int num_rows, int num_blocks,
                                     int max_ctx, int window, int sinks, float scale, int dtype,
                                     int pool_dtype, void* out, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  clear_error();
  if (num_seqs == 0) return KVE_OK;
  KVE_REQUIRE(q && k_layer && v_layer && block_tables && start_pos && out,
              "kve_paged_window_attn: null pointer argument");
  KVE_REQUIRE(window_sizes_ok(num_seqs, q_len, num_q_heads, num_kv_heads, head_dim, max_ctx, window, sinks),
              "kve_paged_window_attn: %d x %d tokens, %d/%d heads of %d (64 or 128), max_ctx %d, "
              "window %d, sinks %d",
              num_seqs, q_len, num_q_heads, num_kv_heads, head_dim, max_ctx, window, sinks);
  KVE_REQUIRE(block_size > 0 && block_size % 16 == 0 && block_size <= (1 << 20),
              "kve_paged_window_attn: block_size %d (a multiple of 16)", block_size);
  KVE_REQUIRE(max_blocks > 0 && num_rows > 0 && num_blocks > 0 &&
                  static_cast<int64_t>(max_blocks) * block_size >= max_ctx,
              "kve_paged_window_attn: %d blocks of %d do not hold max_ctx %d", max_blocks,
              block_size, max_ctx);
  KVE_REQUIRE(static_cast<int64_t>(num_blocks) * num_kv_heads * (block_size / 16) < (1ll << 31),
              "kve_paged_window_attn: pool of %d blocks too large", num_blocks);
  KVE_REQUIRE(scale > 0.0f && scale < INFINITY, "kve_paged_window_attn: scale %g", scale);
  const bool q8 = pool_dtype == KVE_DTYPE_I8 || pool_dtype == KVE_DTYPE_E4M3;
  KVE_REQUIRE((dtype == KVE_DTYPE_BF16 || dtype == KVE_DTYPE_F32) && (q8 || pool_dtype == dtype),
              "kve_paged_window_attn: queries of dtype %d over a pool of dtype %d", dtype, pool_dtype);
  KVE_REQUIRE(!q8 || (k_scale && v_scale), "kve_paged_window_attn: an 8-bit pool needs scales");
  KVE_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_layer) |
                reinterpret_cast<uintptr_t>(v_layer) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
              "kve_paged_window_attn: q, pools and out must be 16-byte aligned");
  const int win = window > 0 ? window : INT32_MAX;
  const WindowCfg c = window_cfg(num_seqs, q_len, num_q_heads, num_kv_heads, head_dim, max_ctx, win,
                                 sinks, step_keys(pool_dtype));
  KVE_REQUIRE(static_cast<int64_t>(num_seqs) * num_kv_heads * c.splits * c.row_groups < (1ll << 31) &&
                  static_cast<int64_t>(num_seqs) * num_q_heads * q_len < (1ll << 31),
              "kve_paged_window_attn: %d x %d tokens too large for one launch", num_seqs, q_len);
  if (workspace_bytes < c.bytes || (c.bytes && !workspace)) {
    set_error("kve_paged_window_attn: workspace %zu bytes, need %zu", workspace_bytes, c.bytes);
    return KVE_EWORKSPACE;
  }
  KVE_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              "kve_paged_window_attn: workspace must be 16-byte aligned");
  WindowArgs a{};
  a.q = q;
  a.k = static_cast<const uint8_t*>(k_layer);
  a.v = static_cast<const uint8_t*>(v_layer);
  a.ks = k_scale;
  a.vs = v_scale;
  a.out = out;
  a.tables = block_tables;
  a.seq_rows = seq_rows;
  a.start_pos = start_pos;
  a.q_lens = q_lens;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + c.ml);
  a.B = num_seqs;
  a.Tq = q_len;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.G = num_q_heads / num_kv_heads;
  a.bs = block_size;
  a.tpb = block_size / 16;
  a.max_blocks = max_blocks;
  a.num_rows = num_rows;
  a.num_blocks = num_blocks;
  a.max_ctx = max_ctx;
  a.window = win;
  a.sinks = sinks;
  a.rw = c.rw;
  a.row_groups = c.row_groups;
  a.chunk = c.chunk;
  a.splits = c.splits;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.g_magic = static_cast<uint32_t>(((1ull << 32) + a.G - 1) / a.G);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (pool_dtype) {
    case KVE_DTYPE_BF16: return launch_window_d<Pool::kBf16, 2>(a, c, head_dim, st);
    case KVE_DTYPE_F32: return launch_window_d<Pool::kF32, 1>(a, c, head_dim, st);
    case KVE_DTYPE_I8:
      return dtype == KVE_DTYPE_BF16 ? launch_window_d<Pool::kInt8, 1>(a, c, head_dim, st)
                                     : launch_window_d<Pool::kInt8, 2>(a, c, head_dim, st);
    default:
      return dtype == KVE_DTYPE_BF16 ? launch_window_d<Pool::kE4m3, 1>(a, c, head_dim, st)
                                     : launch_window_d<Pool::kE4m3, 2>(a, c, head_dim, st);
  }
}
