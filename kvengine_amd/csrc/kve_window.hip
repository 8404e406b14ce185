// Attention over the paged cache with a sliding window and sinks, and over a cache held
// in 8 bits (kve_paged_window_attn). The counterpart in the reference
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
// t G + head). Rows walk the keys they see in steps of 64 (32 in fp32 at head_dim 128): first
// the steps that hold sinks, then those of the window; what lies between is not read. A
// workgroup takes one of two forms:
//  * up to 16 rows (decoding): eight waves with one tile of 16 rows between them, which take
//    the walk's steps in turn; each K/V byte goes into the registers of the one wave that
//    multiplies it, and the eight states are folded through LDS;
//  * more rows (drafts, prompts): four waves, each with one or two tiles of its own, that
//    walk together; a step's K/V comes into LDS once, by direct loads into a ring of 64 KB
//    (two workgroups a CU), RING - 1 steps ahead, and one barrier a step hands it over.
// A long walk is cut into chunks of steps, a workgroup each, that a second launch joins in
// chunk order.
//
// A step. The unit of reading is a fragment: 16 bytes a lane, as the lane needs them for a
// matrix product. A step has parts of 16 NS keys, NS = 4 / bytes of an element (one part in
// 8 bits, two in bf16). Of K, lane (lr, lg) of a part's score product t reads key 4 NS (lr / 4) +
// 4 t + lr % 4, of V channel 16 dt + lr, keys 4 NS lg ... Scores are S^T = K Q^T
// (16x16 matrix products, rows of K on the M side): lane (lr, lg) then holds the scores of
// row lr and keys 4 NS lg + 4 t + i, which are the keys of its V bytes, so P^T goes back
// as an operand of O^T = V^T P^T without leaving the lane. A direct load writes its 64 lanes'
// 16 bytes one after another, so a fragment is read back from LDS without bank conflicts.
//
// Numbers. bf16: products in bf16, P as the sum of two bf16 (16 bits of it; with one, 8 bits, a
// prompt takes 160 us for 190, but its outputs lie 2.16e-3 from 64 bits instead of the 1.62e-3
// that the output's own rounding makes). fp32: fp32 products. 8 bits: codes are exact in fp16, so
// the products are fp16's: q is scaled to the fp16 range by a power of two per row (exact for
// bf16; fp32 as the sum of two fp16, 22 bits), P s_v by a factor per row that follows its largest
// product. For fp32 queries it has two fp16 (22 bits), for bf16 ones one (11 bits): outputs lie
// 1.666e-3 from 64 bits either way at 1000 keys, 1.645e-3 and 1.643e-3 in 16 x 5 rows, and two cost
// 4 % of a decode step (32 long histories 26.2 / 27.3 us) and 12 % of a prompt. Sums, m and l
// are fp32.
//
// Values that a row must not see. A masked score is replaced, not added to, so that nothing
// of its key remains. In V a masked infinity or NaN would be 0 * inf: steps that some
// row sees in part are taken without the non-finite values, which are then added to the rows
// that do see them. Other steps are seen whole by every row. Half of a short walk's steps are
// seen in part, so these are kept cheap: the ends that a step reaches are compared with constants,
// and V is looked over before anything is dropped from it (a tenth of the time of a prompt and of
// 32 x 5 tokens).
//
// What bounds it, at 16 query heads to 2 kv heads of 128 in bf16. A prompt of 4 x 4097 tokens under a
// window of 1024: 182 us in a run of calls, 660 TFLOP/s of the definition's products and half as
// many again for P's second part, the matrix pipes busy 48 % and the vector units 52 % of the time
// and LDS reads 34 %, hardly at once with two waves a SIMD. 32 x 5 new tokens, window 1024: 12.9 us
// and 4.0 for the join, about 1.7 a step (LDS reads, products, softmax, products in series, for
// one of the four waves has no rows there and one half a tile) behind launch, tables and the first
// K/V. 32 int8 histories of 3000 to 8128 tokens, one new token each: 22.7 us (3.8 TB/s) and 4. One
// token of 256 keys: 6.8 us.

#include "kve_gemm.h"
#include "kve_q8.h"

#include <algorithm>
#include <cfloat>
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
  int row_groups, chunk, splits;  // chunk: steps of a workgroup
  float scale_log2;
  uint32_t g_magic;
  int g_shift;
};

constexpr int kKeyWaves = 8;  // waves of a workgroup that share up to 16 rows' steps
constexpr int kMergeThreads = 256;
__host__ __device__ constexpr int win_threads(bool shared) { return shared ? 256 : 64 * kKeyWaves; }
// The maximum of a row that has seen no key. Finite, for -inf less itself is NaN, and no
// score is lower but -inf.
constexpr float kNone = -FLT_MAX;

// Token of row r: r / G for 0 <= r < 2^31. With 2^(s - 1) < G <= 2^s the product with
// ceil(2^(31 + s) / G) is over by r (G - 1) / G / 2^(31 + s) < 1 / G at most.
__device__ __forceinline__ int token_of(const WindowArgs& a, int r) {
  return a.G == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), a.g_magic) >> a.g_shift);
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
  w.p0 = s.start + token_of(a, row0);
  w.p1 = s.start + token_of(a, row1 - 1);
  w.first = w.p0 >= a.window ? (w.p0 - a.window + 1) / SK : 0;
  w.sinks = min((a.sinks + SK - 1) / SK, w.first);
  w.total = w.sinks + w.p1 / SK - w.first + 1;
  return w;
}

// Keys of a step: 64, or what 32 KB of K and V hold (half the ring).
__host__ __device__ constexpr int step_keys(int elem_bytes, int D) {
  return elem_bytes * D == 512 ? 32 : 64;
}

// ---- element types ----------------------------------------------------------------

template <Pool P, int D>
struct PoolOf {
  static constexpr int ES = P == Pool::kF32 ? 4 : P == Pool::kBf16 ? 2 : 1;
  static constexpr bool Q8B = ES == 1;
  static constexpr int NS = 4 / ES;                  // 16-key tiles of a part of a step
  static constexpr int U = step_keys(ES, D) / (16 * NS);  // parts
  static constexpr int NT = NS * U, SK = 16 * NT;    // tiles and keys of a step
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

// Whether some value of four 16-byte vectors is not finite.
template <Pool P>
__device__ __forceinline__ bool any_nonfinite(const u32x4 (&x)[4]) {
  uint32_t top = 0;  // bf16: the largest magnitudes of the halves; fp32: of all; e4m3: flags
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t w = x[i >> 2][i & 3];
    if constexpr (P == Pool::kBf16) {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, w & 0x7fff7fffu),
                                                                   __builtin_bit_cast(u16x2, top)));
    } else if constexpr (P == Pool::kF32) {
      top = max(top, w & 0x7fffffffu);
    } else {
      top |= (w & 0x7f7f7f7fu) + 0x01010101u;
    }
  }
  if constexpr (P == Pool::kBf16) return ((top + 0x00800080u) & 0x80008000u) != 0;
  if constexpr (P == Pool::kF32) return top >= 0x7f800000u;
  return (top & 0x80808080u) != 0;
}

// The non-finite values of 16 bytes set to 0.
template <Pool P>
__device__ __forceinline__ void drop_nonfinite(u32x4& x) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (P == Pool::kBf16)
      x[w] &= ~(((((x[w] & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu);
    else if constexpr (P == Pool::kF32)
      x[w] = (x[w] & 0x7f800000u) == 0x7f800000u ? 0u : x[w];
    else
      x[w] &= ~(((((x[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu);
  }
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

constexpr int kRingBytes = 64 * 1024;

// How far a row's maximum may lag behind its scores (in powers of 2) before its state is
// rescaled: P stays below 2^8.
constexpr float kLag = 8.0f;

// QP: fp16 parts that q is taken as over 8-bit pools (1: bf16 queries, 2: fp32; else 1).
// PP: 16-bit parts of P (fp32 pools: 1, whole).
template <Pool P, int QP, int PP, int D, int MT, bool SHARED>
__global__ __launch_bounds__(win_threads(SHARED)) __attribute__((amdgpu_waves_per_eu(2, 2))) void window_attn_kernel(WindowArgs a) {
  using X = PoolOf<P, D>;
  constexpr int ES = X::ES, NS = X::NS, U = X::U, NT = X::NT, SK = X::SK, SP = 16 * NS;
  constexpr bool Q8B = X::Q8B, F32 = P == Pool::kF32;
  constexpr bool QBF = P == Pool::kBf16 || (Q8B && QP == 1);  // q and out in bf16
  constexpr int KW = SHARED ? 1 : kKeyWaves;
  constexpr int ROWS = 16 * MT * (SHARED ? 4 : 1);
  constexpr int NJ = D * ES / 64;  // fragments of a K row
  constexpr int DT = D / 16;
  constexpr int NF = F32 ? D / 16 : D / 32;  // fragments of q
  constexpr int FRAGS = U * 2 * DT;          // of a step: each part's K (NS NJ = DT), then its V
  constexpr int LPW = FRAGS / 4;             // a wave's loads of a shared step
  static_assert(NS * NJ == DT, "as many fragments of K as of V");
  constexpr int RING = kRingBytes / (FRAGS * 1024);
  constexpr int BATCH = 64 / NT;  // steps whose block ids a wave holds
  extern __shared__ float sm[];

  const int tid = threadIdx.x, l = tid & 63, lr = l & 15, lg = l >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  // The last rows of all sequences come first: their walks are the longest, and what is left
  // at the end is short (4 % of a prompt of 4 x 4097 tokens).
  int u = blockIdx.x;
  const int c = u % a.splits;
  u /= a.splits;
  const int kvh = u % a.Hkv;
  u /= a.Hkv;
  const int b = u % a.B, rg = a.row_groups - 1 - u / a.B;
  const WinSeq s = win_seq(a, b);
  const int R = a.G * s.T, g0 = rg * ROWS;
  if (g0 >= R) return;
  const Walk w = walk_of<SK>(a, s, g0, min(R, g0 + ROWS));
  const int chunks = cdiv(w.total, a.chunk);
  if (c >= chunks) return;
  // the wave's rows, and its steps at, at + KW, ... (n of them)
  const int row0 = SHARED ? g0 + wid * 16 * MT : g0, row1 = min(R, row0 + 16 * MT);
  const int kw = SHARED ? 0 : wid, at = c * a.chunk + kw;
  const int n = cdiv(max(min(w.total, (c + 1) * a.chunk) - at, 0), KW);
  const bool active = row0 < R;
  const int p0 = active ? s.start + token_of(a, row0) : w.p0;
  const int p1 = active ? s.start + token_of(a, row1 - 1) : w.p1;

  // q as it lies in memory: the lane's channels of row lr of each tile, in the order of its
  // K fragments. Asked for first, for behind the first K and V it would wait for all of them.
  constexpr int QV = Q8B && !QBF ? 2 : 1;  // vectors of a fragment of 8 channels
  u32x4 qf[MT][QP][NF], qraw[MT][Q8B ? NF * QV : 1];
  int qpos[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = min(row0 + mt * 16 + lr, R - 1);
    const int t = token_of(a, r), h = kvh * a.G + r - t * a.G;
    qpos[mt] = s.start + t;
    const size_t qat = ((static_cast<size_t>(b) * a.Tq + t) * a.Hq + h) * D;
    if constexpr (!Q8B) {
      const uint8_t* qp = static_cast<const uint8_t*>(a.q) + qat * ES + lg * 16;
#pragma unroll
      for (int j = 0; j < NF; ++j) qf[mt][0][j] = *reinterpret_cast<const u32x4*>(qp + j * 64);
    } else {
      // channels 64 j + 16 lg + 8 f .. of fragment 2 j + f
      const uint8_t* qp = static_cast<const uint8_t*>(a.q) + (qat + lg * 16) * (2 * QV);
#pragma unroll
      for (int x = 0; x < NF * QV; ++x)
        qraw[mt][x] = *reinterpret_cast<const u32x4*>(
            qp + ((x / QV >> 1) * 64 + (x / QV & 1) * 8) * (2 * QV) + x % QV * 16);
    }
  }

  // the first steps' block ids
  const int32_t* table = a.tables + static_cast<size_t>(s.row) * a.max_blocks;
  const int last_tile = w.p1 >> 4;
  const auto tile_of = [&](int i) {  // lane: tile l % NT of step i + l / NT (past the last: it again)
    const int st = w.step(at + min(i + l / NT, n - 1) * KW);
    return min(st * NT + l % NT, last_tile);
  };
  const auto read_table = [&](int i) {  // (within the table: start + T <= max_ctx <= its blocks)
    const int tile = tile_of(i);
    return table[a.tpb == 1 ? tile : tile / a.tpb];
  };
  // Where the tile is, in units of 16 bytes from the start of the K and the V pool (the host
  // holds pools below 2^36 bytes), and its (block, head).
  struct Place {
    uint32_t k, v;
    int bh;
  };
  const auto place = [&](int blk, int i) {
    const int part = a.tpb == 1 ? 0 : tile_of(i) % a.tpb;
    Place x;
    x.bh = (static_cast<unsigned>(blk) < static_cast<unsigned>(a.num_blocks) ? blk : 0) * a.Hkv + kvh;
    const uint32_t first = static_cast<uint32_t>(x.bh) * static_cast<uint32_t>(a.bs * D * ES / 16);
    x.k = first + part * (D * ES);
    x.v = first + part * ES;
    return x;
  };
  Place ids{}, ids1{};  // of the batch, of the next one
  int raw1 = 0;         // the next batch's table entries
  float ksl = 0, vsl = 0, ks1 = 0, vs1 = 0;  // the lane's tile's scales, the next batch's
  if (n > 0) {
    ids = place(read_table(0), 0);
    if (n > BATCH) raw1 = read_table(BATCH);
  }

  // fragments: where the lane reads within a tile
  const int kk = 4 * NS * (lr >> 2) + (lr & 3), vk = 4 * NS * lg;
  const size_t vrow = static_cast<size_t>(a.bs) * ES;
  const uint8_t* klane = a.k + (kk & 15) * D * ES + lg * 16;
  const uint8_t* vlane = a.v + lr * vrow + (vk & 15) * ES;
  // the lane's K or V address of part p of step i; `now`: the step whose batch `ids` is
  const auto k_at = [&](int i, int p, int now) {
    const int id = __shfl(static_cast<int>(i / BATCH == now / BATCH ? ids.k : ids1.k),
                          i % BATCH * NT + p * NS + (kk >> 4));
    return klane + static_cast<uint64_t>(static_cast<uint32_t>(id)) * 16;
  };
  const auto v_at = [&](int i, int p, int now) {
    const int id = __shfl(static_cast<int>(i / BATCH == now / BATCH ? ids.v : ids1.v),
                          i % BATCH * NT + p * NS + (vk >> 4));
    return vlane + static_cast<uint64_t>(static_cast<uint32_t>(id)) * 16;
  };

  u32x4 kf[U][SHARED ? 1 : DT], vf[U][SHARED ? 1 : DT];
  uint8_t* ring = reinterpret_cast<uint8_t*>(sm);
  const auto load_k = [&](int i, int now) {
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const uint8_t* at = k_at(i, p, now);
#pragma unroll
      for (int f = 0; f < DT; ++f)
        kf[p][f] = *reinterpret_cast<const u32x4*>(at + f / NJ * (4 * D * ES) + f % NJ * 64);
    }
  };
  const auto load_v = [&](int i, int now) {
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const uint8_t* at = v_at(i, p, now);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        vf[p][dt] = *reinterpret_cast<const u32x4*>(at + dt * 16 * vrow);
    }
  };
  // Waves 0 and 1 load a shared step's K fragments, 2 and 3 its V's: what they read is
  // settled here, for the loop.
  const bool is_k = wid < 2;
  const int f0 = (wid & 1) * (DT / 2);
  const uint8_t* mine = is_k ? klane : vlane;
  const int my_tile = is_k ? kk >> 4 : vk >> 4;
  uint32_t skip[DT / 2];  // from the lane's address to each fragment
#pragma unroll
  for (int x = 0; x < DT / 2; ++x)
    skip[x] = is_k ? (f0 + x) / NJ * (4 * D * ES) + (f0 + x) % NJ * 64
                   : static_cast<uint32_t>((f0 + x) * 16 * vrow);
  const auto stage = [&](int i, int now) {
    const bool here = i / BATCH == now / BATCH;
    const int id = static_cast<int>(is_k ? (here ? ids.k : ids1.k) : (here ? ids.v : ids1.v));
    uint8_t* to = ring + (i % RING) * (FRAGS * 1024) + ((is_k ? 0 : DT) + f0) * 1024;
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const uint32_t off = __shfl(id, i % BATCH * NT + p * NS + my_tile);
      const uint8_t* at = mine + static_cast<uint64_t>(off) * 16;
#pragma unroll
      for (int x = 0; x < DT / 2; ++x)
        __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(at + skip[x]),
                                         (__attribute__((address_space(3))) void*)(to + (2 * DT * p + x) * 1024),
                                         16, 0, 0);
    }
  };
  if (SHARED) {
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
      if (i < n) stage(i, 0);
  } else if (n > 0) {
    load_k(0, 0);
    load_v(0, 0);
  }
  if (Q8B && n > 0) {
    ksl = a.ks[ids.bh];
    vsl = a.vs[ids.bh];
  }

  float rf[MT];  // score -> exponent of 2
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    rf[mt] = a.scale_log2;
    if constexpr (Q8B) {
      float x[NF][8];
      float top = 0.0f;
#pragma unroll
      for (int f = 0; f < NF; ++f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (QBF)
            x[f][e] = __uint_as_float(e & 1 ? qraw[mt][f][e >> 1] & 0xffff0000u : qraw[mt][f][e >> 1] << 16);
          else
            x[f][e] = __uint_as_float(qraw[mt][2 * f + (e >> 2)][e & 3]);
          top = fmaxf(top, fabsf(x[f][e]));
        }
      }
      top = max_across_groups(top);
      // the row's largest value to [2^13, 2^14): what falls below fp16's steps of 2^-24
      // there is below 2^-37 of it
      const int ex = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
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

  f32x4 acc[MT][DT];
  float m[MT], lsum[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = f32x4{0, 0, 0, 0};
    m[mt] = kNone;
    lsum[mt] = 0.0f;
  }
  // 8-bit: a row's acc is in units of ref 2^-14, ref above every P s_v that it has met, in units
  // of its present maximum. By row and from P, not from the scales of the walk's blocks: a
  // block that a row does not see, or gives no weight, takes no bits from the others.
  float ref[MT], per_ref[MT];  // per_ref = 2^14 / ref
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    ref[mt] = kMinScale;
    per_ref[mt] = 0x1p14f / kMinScale;
  }

  for (int i = 0; i < n; ++i) {
    if (n > BATCH && i % (BATCH / 2) == 0) {
      if (i % BATCH == 0) {
        if (i > 0) {
          ids = ids1;
          ksl = ks1;
          vsl = vs1;
          if (i + BATCH < n) raw1 = read_table(i + BATCH);
        }
      } else if (i + BATCH / 2 < n) {
        ids1 = place(raw1, i + BATCH / 2);
        if (Q8B) {
          ks1 = a.ks[ids1.bh];
          vs1 = a.vs[ids1.bh];
        }
      }
    }
    const uint8_t* here = ring + (i % RING) * (FRAGS * 1024) + l * 16;
    if (SHARED) {
      // step i has landed for every wave, and all are done with step i - 1, whose place
      // takes step i + RING - 1
      barrier_after_chunks<LPW, RING - 2>(min(RING - 2, n - 1 - i));
      if (i + RING - 1 < n) stage(i + RING - 1, i);
    }
    const int k0 = w.step(at + i * KW) * SK;
    // (a wave whose rows see nothing of a shared step sits it out)
    if (SHARED && (!active || k0 > p1 || (k0 + SK - 1 <= p0 - a.window && k0 >= a.sinks))) continue;
    // Fragments are taken NT (of K) and four (of V) at a time, the next ones on their way from
    // LDS while some are multiplied (the compiler left to itself reads each right before its
    // products and waits for it), and products that add to one sum are kept apart.
    const auto k_frag = [&](int j, int t) {
      const int f = t % NS * NJ + j;
      return SHARED ? *reinterpret_cast<const u32x4*>(here + (2 * DT * (t / NS) + f) * 1024)
                    : kf[t / NS][SHARED ? 0 : f];
    };
    const auto v_frag = [&](int g, int x) {
      const int dt = g % (DT / 4) * 4 + x, p = g / (DT / 4);
      return SHARED ? *reinterpret_cast<const u32x4*>(here + (2 * DT * p + DT + dt) * 1024)
                    : vf[p][SHARED ? 0 : dt];
    };
    f32x4 sc[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int t = 0; t < NT; ++t) sc[mt][t] = f32x4{0, 0, 0, 0};
    }
    u32x4 kn[NT], vn[4];
#pragma unroll
    for (int t = 0; t < NT; ++t) kn[t] = k_frag(0, t);
    // (a wave in its products goes before one in its softmax: 1 % of a prompt)
    if (SHARED) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      u32x4 kc[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) kc[t] = kn[t];
      if (j + 1 < NJ) {
#pragma unroll
        for (int t = 0; t < NT; ++t) kn[t] = k_frag(j + 1, t);
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) vn[x] = v_frag(0, x);
      }
      if (SHARED) __builtin_amdgcn_sched_barrier(0);
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              sc[mt][t] = mfma16x16x4_f32(__uint_as_float(kc[t][e]), __uint_as_float(qf[mt][0][j][e]),
                                          sc[mt][t]);
          }
        }
      } else if constexpr (Q8B) {
        u32x4 f[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) codes_to_frags<P>(kc[t], f[t]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int q = 0; q < QP; ++q) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
                sc[mt][t] = mfma16x16x32_f16(f[t][e], qf[mt][q][2 * j + e], sc[mt][t]);
            }
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) sc[mt][t] = mfma16x16x32_bf16(kc[t], qf[mt][0][j], sc[mt][t]);
        }
      }
      if (SHARED) __builtin_amdgcn_sched_barrier(0);
    }
    if (SHARED) __builtin_amdgcn_s_setprio(0);
    if (SHARED) __asm__ volatile("" ::: "memory");  // the first of V stays ahead of the softmax
    if (!SHARED && i + 1 < n) load_k(i + 1, i);
    float ks = 1.0f, vs = 1.0f;
    if constexpr (Q8B) {
      ks = __shfl(ksl, i % BATCH * NT + lg);
      vs = __shfl(vsl, i % BATCH * NT + lg);
    }
    // seen whole by every row of the wave
    const bool whole = k0 + SK - 1 <= p0 && (k0 > p1 - a.window || k0 + SK <= a.sinks);
    u32x4 pf[MT][U][PP][Q8B ? 2 : 1];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float f = Q8B ? rf[mt] * ks : rf[mt];
      if (!whole) {
        if constexpr (Q8B) {  // the exponents themselves: a masked key's scale may be no number
#pragma unroll
          for (int x = 0; x < 4 * NT; ++x) sc[mt][x >> 2][x & 3] *= f;
          f = 1.0f;
        }
        // key k0 + 4 NS lg + (a constant of x) against the ends of what the row sees, the
        // window's last and its first, each where the step reaches it
        const int at = k0 + 4 * NS * lg;
        if (k0 + SK - 1 > p0) {
          const int last = qpos[mt] - at;
#pragma unroll
          for (int x = 0; x < 4 * NT; ++x)
            sc[mt][x >> 2][x & 3] = x / (4 * NS) * SP + x % (4 * NS) <= last ? sc[mt][x >> 2][x & 3] : -INFINITY;
        }
        if (k0 <= p1 - a.window) {
          const int before = qpos[mt] - a.window - at, sunk = a.sinks - at;
#pragma unroll
          for (int x = 0; x < 4 * NT; ++x) {
            const int y = x / (4 * NS) * SP + x % (4 * NS);
            sc[mt][x >> 2][x & 3] = (y > before) | (y < sunk) ? sc[mt][x >> 2][x & 3] : -INFINITY;
          }
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < 4 * NT; ++x) top = fmaxf(top, sc[mt][x >> 2][x & 3]);
      const float own = top;  // of the lane's keys, in 8 bits those of one tile
      top = max_across_groups(top * f);
      const bool grow = top > m[mt] + kLag;
      if (__any(grow)) {
        const float to = grow ? top : m[mt], al = __builtin_amdgcn_exp2f(m[mt] - to);
        m[mt] = to;
        lsum[mt] *= al;
        if constexpr (Q8B) {
          ref[mt] *= al;
        } else {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= al;
        }
      }
      float unit = 1.0f;
      if constexpr (Q8B) {
        // the lane's largest P s_v; P counts as 2^-100 at the least, which keeps s_v / ref in range
        const float p = __builtin_amdgcn_exp2f(fmaf(own, f, -m[mt]));
        const bool number = fabsf(vs) < INFINITY;  // (what is none goes its own way)
        const float most = max_across_groups(p > 0.0f && number ? fabsf(vs) * fmaxf(p, 0x1p-100f) : 0.0f);
        if (__any(grow || most >= ref[mt])) {
          const float was = ref[mt];
          ref[mt] = fminf(fmaxf(most >= was ? 2.0f * most : was, kMinScale), 0x1p127f);
          per_ref[mt] = 0x1p14f / ref[mt];
          const float al = was / ref[mt];
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= al;
        }
        unit = p > 0.0f || !number ? vs * per_ref[mt] : 0.0f;
      }
      float x[4 * NT];
      float add = 0.0f;
#pragma unroll
      for (int e = 0; e < 4 * NT; ++e) {
        x[e] = __builtin_amdgcn_exp2f(fmaf(sc[mt][e >> 2][e & 3], f, -m[mt]));
        add += x[e];
      }
      lsum[mt] += add;
      if constexpr (Q8B) {
        // (0 * s_v of a block whose scale is no number stays 0)
#pragma unroll
        for (int e = 0; e < 4 * NT; ++e) x[e] = whole || x[e] != 0.0f ? x[e] * unit : 0.0f;
      }
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4 * NT; ++e) pf[mt][e >> 2][0][0][e & 3] = __float_as_uint(x[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 2 * NT; ++e) {
#pragma unroll
          for (int p = 0; p < PP; ++p) {
            uint32_t h;
            if constexpr (Q8B)
              h = p + 1 < PP ? split_f16x2(x[2 * e], x[2 * e + 1]) : pack_f16x2(x[2 * e], x[2 * e + 1]);
            else
              h = p + 1 < PP ? split_bf16x2(x[2 * e], x[2 * e + 1]) : pack_bf16x2(x[2 * e], x[2 * e + 1]);
            pf[mt][e / (2 * NS)][p][e % (2 * NS) >> 2][e & 3] = h;
          }
        }
      }
    }
    bool dropped = false;
    if (SHARED) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int g = 0; g < U * DT / 4; ++g) {
      const int p = g / (DT / 4), d0 = g % (DT / 4) * 4;
      u32x4 vc[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) vc[x] = vn[x];
      if (g + 1 < U * DT / 4) {
#pragma unroll
        for (int x = 0; x < 4; ++x) vn[x] = v_frag(g + 1, x);
      }
      if (SHARED) __builtin_amdgcn_sched_barrier(0);
      if constexpr (P != Pool::kInt8) {
        if (!whole && __builtin_expect(__any(any_nonfinite<P>(vc)), 0)) {
          dropped = true;
#pragma unroll
          for (int x = 0; x < 4; ++x) drop_nonfinite<P>(vc[x]);
        }
      }
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              acc[mt][d0 + x] = mfma16x16x4_f32(__uint_as_float(vc[x][e]),
                                                __uint_as_float(pf[mt][p][0][0][e]), acc[mt][d0 + x]);
          }
        }
      } else if constexpr (Q8B) {
        u32x4 f[4][2];
#pragma unroll
        for (int x = 0; x < 4; ++x) codes_to_frags<P>(vc[x], f[x]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int q = 0; q < PP; ++q) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
                acc[mt][d0 + x] = mfma16x16x32_f16(f[x][e], pf[mt][p][q][e], acc[mt][d0 + x]);
            }
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < PP; ++q) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              acc[mt][d0 + x] = mfma16x16x32_bf16(vc[x], pf[mt][p][q][0], acc[mt][d0 + x]);
          }
        }
      }
      if (SHARED) __builtin_amdgcn_sched_barrier(0);
    }
    if (SHARED) __builtin_amdgcn_s_setprio(0);
    if (dropped) {
      // rare: the step's keys one by one, their non-finite values to the rows that see them
#pragma unroll 1
      for (int x = 0; x < SK; ++x) {
        const int key = k0 + x;
        if (key > p1) break;
        const uint32_t off = __shfl(static_cast<int>(ids.v), i % BATCH * NT + (x >> 4));
        const uint8_t* p = a.v + static_cast<uint64_t>(off) * 16 + 4 * lg * vrow + (x & 15) * ES;
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
    if (!SHARED && i + 1 < n) load_v(i + 1, i);
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    lsum[mt] = sum_across_groups(lsum[mt]);
    if constexpr (Q8B) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= ref[mt] * 0x1p-14f;
    }
  }

  if constexpr (!SHARED) {
    // the waves' states, in order, into the first's
    constexpr int WAVE = MT * (DT * 256 + 32);  // floats a wave leaves
    float* mine = sm + (wid - 1) * WAVE;
    if (wid > 0) {
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
    if (wid > 0) return;
#pragma unroll
    for (int o = 0; o < KW - 1; ++o) {
      const float* other = sm + o * WAVE;
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
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = row0 + mt * 16 + lr;
    if (r >= R) continue;
    if (chunks == 1) {
      const int t = token_of(a, r), h = kvh * a.G + r - t * a.G;
      const size_t to = ((static_cast<size_t>(b) * a.Tq + t) * a.Hq + h) * D + 4 * lg;
      const float inv = 1.0f / lsum[mt];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f32x4 y = acc[mt][dt] * inv;
        if constexpr (QBF)
          *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + to + dt * 16) =
              u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        else
          *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + to + dt * 16) = y;
      }
    } else {
      const size_t slot =
          ((static_cast<size_t>(b) * a.Hkv + kvh) * a.splits + c) * a.row_groups * ROWS + r;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<f32x4*>(a.part_o + slot * D + dt * 16 + 4 * lg) = acc[mt][dt];
      if (lg == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = float2{m[mt], lsum[mt]};
    }
  }
}

// Rows whose walk has several chunks: the chunks' states joined in chunk order, a wave
// per row, D / 64 channels a lane. The first chunks are asked for before the row's walk
// is known (the workspace holds them whatever it is), the others four at a time.
template <int SK, int D, bool OUT_BF16>
__global__ __launch_bounds__(kMergeThreads) void window_merge_kernel(WindowArgs a, int unit_rows) {
  constexpr int N = D / 64, AHEAD = 4;
  struct alignas(4 * N) Vec { float v[N]; };
  const int l = threadIdx.x & 63;
  const int rmax = a.G * a.Tq;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * (kMergeThreads / 64) + (threadIdx.x >> 6);
  if (u >= static_cast<int64_t>(a.B) * a.Hkv * rmax) return;
  const int r = static_cast<int>(u % rmax), bh = static_cast<int>(u / rmax);
  const int b = bh / a.Hkv, kvh = bh - b * a.Hkv;
  const size_t per = static_cast<size_t>(a.row_groups) * unit_rows;
  const size_t slot0 = static_cast<size_t>(bh) * a.splits * per + r;
  float2 ml[AHEAD];
  Vec po[AHEAD];
  const auto load = [&](int c0) {
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) {
      const size_t slot = slot0 + min(c0 + x, a.splits - 1) * per;
      ml[x] = *reinterpret_cast<const float2*>(a.part_ml + slot * 2);
      po[x] = *reinterpret_cast<const Vec*>(a.part_o + slot * D + l * N);
    }
  };
  load(0);
  const WinSeq s = win_seq(a, b);
  const int R = a.G * s.T;
  if (r >= R) return;
  const int row0 = r / unit_rows * unit_rows;
  const Walk w = walk_of<SK>(a, s, row0, min(R, row0 + unit_rows));
  const int chunks = cdiv(w.total, a.chunk);
  if (chunks == 1) return;
  float m = kNone, sum = 0.0f;
  Vec o{};
  for (int c0 = 0; c0 < chunks; c0 += AHEAD) {
    if (c0) load(c0);
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) {
      if (c0 + x >= chunks) break;
      const float to = fmaxf(m, ml[x].x), al = __builtin_amdgcn_exp2f(m - to),
                  be = __builtin_amdgcn_exp2f(ml[x].x - to);
      m = to;
      sum = sum * al + ml[x].y * be;
#pragma unroll
      for (int e = 0; e < N; ++e) o.v[e] = o.v[e] * al + po[x].v[e] * be;
    }
  }
  const int t = token_of(a, r), h = kvh * a.G + r - t * a.G;
  const size_t to = ((static_cast<size_t>(b) * a.Tq + t) * a.Hq + h) * D + l * N;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = o.v[e] / sum;
    if constexpr (OUT_BF16) static_cast<uint16_t*>(a.out)[to + e] = f32_to_bf16(y);
    else static_cast<float*>(a.out)[to + e] = y;
  }
}

// ---- launch -------------------------------------------------------------------------

// Waves that a launch should have before walks are cut: eight per compute unit.
constexpr int kFillWaves = 2048;
// Workgroups from which on a wave takes two tiles of rows: two for each compute unit.
constexpr int kTwoTiles = 512;
// Tokens of history by whose whole numbers the cut of a walk follows max_ctx.
constexpr int kCtxStep = 256, kCtxLeast = 1024;

struct WindowCfg {
  int mt, rows, row_groups, chunk, splits;  // mt 0: up to 16 rows
  size_t ml, bytes;  // offset of part_ml, the workspace's size
};

// Walks are not cut below `least` steps, where a chunk's own start and its part of the
// join outweigh the steps it takes over: more than 16 rows, 1 / 2 / 4 / 8 steps, bf16 (32 x 5
// tokens, window 1024) 16.8 / 16.9 / 17.1 / 20.0 us, 8-bit (16 x 5) 19.5 / 19.5 / 18.0 / 22.5, fp32
// pools, bound by their products, 11.2 / 12.9 / 17.8 / 23.1. Up to 16 rows, 8 / 16 / 32 steps: 8 long
// histories in bf16 17.9 / 20.5 / 28.3, 32 under a window of 1024 14.8 / 19.2 / 17.7; where
// all waves are done in two turns, the join costs more than it gains (1000 keys 9.5 us, 8.4
// in one piece). Eight waves for four: 32 long 8-bit histories 28.3 -> 25.9 us.
// Two tiles a wave halve the LDS reads per product and pay where workgroups of twice the rows
// still fill the chip, two a compute unit, and few of their rows are empty. 1 / 2 tiles, window
// 1024, 16 query heads of 128, by workgroups of 128 rows: prompts in bf16 152 18 / 32 us, 258 36 /
// 40, 376 39 / 43, 516 55 / 51, 656 58 / 49, 1032 103 / 89, 2056 227 / 188; 8-bit 258 42 / 51, 376
// 48 / 54, 516 71 / 60, 1032 123 / 105, 2056 270 / 212; 9 tokens a sequence in bf16 128 30 / 31, 192
// 36 / 43, 384 57 / 59, 512 75 / 63, 1024 147 / 115 (at 96 alone, where one round of workgroups is as
// long as the longest walk, 28 / 26). With 264 rows, which take 384 for 320, 768 workgroups 84 / 93,
// with 520, 640 for 576, 640 workgroups 77 / 84. fp32 queries, bound by products or registers, keep
// one (prompt of 1025 242 / 275 us). So many workgroups are never cut.
static WindowCfg window_cfg(int B, int Tq, int Hq, int Hkv, int D, int max_ctx, int window,
                            int sinks, int elem_bytes, bool f32) {
  WindowCfg c{};
  const int R = Hq / Hkv * Tq, sk = step_keys(elem_bytes, D);
  const int t64 = cdiv(R, 64), t128 = cdiv(R, 128);  // workgroups of 64 rows, of 128
  const bool two = !f32 && R > 64 && static_cast<int64_t>(B) * Hkv * t128 >= kTwoTiles &&
                   2 * t128 <= t64 + t64 / 16;
  c.mt = R <= 16 ? 0 : two ? 2 : 1;
  c.rows = c.mt ? 64 * c.mt : 16;
  c.row_groups = cdiv(R, c.rows);
  // the longest walk: the window of a workgroup's first query to its last, and the sinks; or all keys
  const int64_t in_window = (static_cast<int64_t>(window) + cdiv(c.rows, Hq / Hkv) + 1) / sk + 2 +
                            (static_cast<int64_t>(sinks) + sk - 1) / sk;
  // max_ctx decides where walks are cut by what it is in whole kCtxStep: a pass gives the same bits
  // under every bound from one to the next
  // (one sequence in bf16, as replayed iterations are, also under every bound up to kCtxLeast)
  const int bound = B == 1 && !f32 ? std::max(max_ctx, kCtxLeast) : max_ctx;
  const int64_t in_all = static_cast<int64_t>(cdiv(bound, kCtxStep)) * (kCtxStep / sk);
  const int64_t longest = std::min(in_window, in_all);
  const int waves = c.mt == 0 ? kKeyWaves : 4;
  int64_t least = c.mt == 0 ? kKeyWaves : elem_bytes == 4 ? 1 : 4;
  if (c.mt == 0 && (in_window <= 2 * kKeyWaves + 1 || in_all <= 2 * kKeyWaves)) least = longest;
  const int64_t units = static_cast<int64_t>(B) * Hkv * c.row_groups;
  const int64_t want = std::max<int64_t>(1, kFillWaves / waves / units);
  int64_t chunk = std::max<int64_t>((longest + want - 1) / want, least);
  if (c.mt == 0) chunk = (chunk + kKeyWaves - 1) / kKeyWaves * kKeyWaves;
  const int64_t steps = std::min<int64_t>(in_window, cdiv(max_ctx, sk));
  c.splits = static_cast<int>((steps + chunk - 1) / chunk);
  c.chunk = static_cast<int>(chunk);
  if (c.splits > 1) {
    const size_t slots = static_cast<size_t>(B) * Hkv * c.splits * c.row_groups * c.rows;
    c.ml = slots * D * sizeof(float);
    c.bytes = c.ml + slots * 2 * sizeof(float);
  }
  return c;
}

template <Pool P, int QP, int PP, int D, int MT, bool SHARED>
static void launch_walk(const WindowArgs& a, hipStream_t st) {
  const int64_t grid = static_cast<int64_t>(a.B) * a.Hkv * a.splits * a.row_groups;
  const size_t lds = SHARED ? kRingBytes : (kKeyWaves - 1) * MT * (D * 16 + 32) * sizeof(float);
  hipLaunchKernelGGL((window_attn_kernel<P, QP, PP, D, MT, SHARED>), dim3(static_cast<unsigned>(grid)),
                     dim3(win_threads(SHARED)), lds, st, a);
}

template <Pool P, int QP, int PP, int D>
static int launch_window(const WindowArgs& a, const WindowCfg& c, hipStream_t st) {
  constexpr bool kTwo = P != Pool::kF32 && QP == 1;  // bf16 queries
  if (c.mt == 0) launch_walk<P, QP, PP, D, 1, false>(a, st);
  else if (c.mt == 1) launch_walk<P, QP, PP, D, 1, true>(a, st);
  else if constexpr (kTwo) launch_walk<P, QP, PP, D, 2, true>(a, st);
  if (c.splits > 1) {
    constexpr bool bf = P == Pool::kBf16 || (PoolOf<P, D>::Q8B && QP == 1);
    const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * a.G * a.Tq;
    hipLaunchKernelGGL((window_merge_kernel<PoolOf<P, D>::SK, D, bf>),
                       dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(kMergeThreads), 0, st, a, c.rows);
  }
  return check_launch("kve_paged_window_attn");
}

template <Pool P, int QP, int PP>
static int launch_window_d(const WindowArgs& a, const WindowCfg& c, int D, hipStream_t st) {
  return D == 64 ? launch_window<P, QP, PP, 64>(a, c, st) : launch_window<P, QP, PP, 128>(a, c, st);
}

static int elem_bytes(int pool_dtype) {
  return pool_dtype == KVE_DTYPE_F32 ? 4 : pool_dtype == KVE_DTYPE_BF16 ? 2 : 1;
}

static bool window_sizes_ok(int B, int Tq, int Hq, int Hkv, int D, int max_ctx, int window, int sinks) {
  return B > 0 && Tq > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && (D == 64 || D == 128) &&
         max_ctx > 0 && max_ctx <= (1 << 30) && window >= 0 && sinks >= 0 &&
         static_cast<int64_t>(Hq / Hkv) * Tq < (1 << 30);
}

}  // namespace kve

using namespace kve;

extern "C" size_t kve_window_workspace_bytes(int num_seqs, int q_len, int num_q_heads,
                                             int num_kv_heads, int head_dim, int max_ctx,
                                             int window, int sinks, int dtype, int pool_dtype) {
  if (!window_sizes_ok(num_seqs, q_len, num_q_heads, num_kv_heads, head_dim, max_ctx, window, sinks))
    return 0;
  return window_cfg(num_seqs, q_len, num_q_heads, num_kv_heads, head_dim, max_ctx,
                    window > 0 ? window : INT32_MAX, sinks, elem_bytes(pool_dtype),
                    dtype == KVE_DTYPE_F32)
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
  // (offsets in units of 16 bytes are 32-bit, and so is a block's number times the heads)
  KVE_REQUIRE(static_cast<int64_t>(num_blocks) * num_kv_heads < (1ll << 31) &&
                  static_cast<int64_t>(num_blocks) * num_kv_heads * (block_size / 16) * head_dim *
                          elem_bytes(pool_dtype) <
                      (1ll << 32),
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
                                 sinks, elem_bytes(pool_dtype), dtype == KVE_DTYPE_F32);
  // (a launch has below 2^32 threads: 512 a workgroup, 64 a row in the join)
  KVE_REQUIRE(static_cast<int64_t>(num_seqs) * num_kv_heads * c.splits * c.row_groups < (1ll << 23) &&
                  static_cast<int64_t>(num_seqs) * num_q_heads * q_len < (1ll << 26),
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
  // (no more than there are keys: the walk rounds them up to whole steps in 32 bits)
  a.sinks = std::min(sinks, max_ctx);
  a.row_groups = c.row_groups;
  a.chunk = c.chunk;
  a.splits = c.splits;
  a.scale_log2 = scale * 1.44269504088896340736f;
  int s = 1;
  while ((1ll << s) < a.G) ++s;
  a.g_magic = static_cast<uint32_t>(((1ull << (31 + s)) + a.G - 1) / a.G);
  a.g_shift = s - 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (pool_dtype) {
    case KVE_DTYPE_BF16: return launch_window_d<Pool::kBf16, 1, 2>(a, c, head_dim, st);
    case KVE_DTYPE_F32: return launch_window_d<Pool::kF32, 1, 1>(a, c, head_dim, st);
    case KVE_DTYPE_I8:
      return dtype == KVE_DTYPE_BF16 ? launch_window_d<Pool::kInt8, 1, 1>(a, c, head_dim, st)
                                     : launch_window_d<Pool::kInt8, 2, 2>(a, c, head_dim, st);
    default:
      return dtype == KVE_DTYPE_BF16 ? launch_window_d<Pool::kE4m3, 1, 1>(a, c, head_dim, st)
                                     : launch_window_d<Pool::kE4m3, 2, 2>(a, c, head_dim, st);
  }
}
