// New K/V rows into a cache held in 8 bits (kve_kv_write_q8): the paged scatter of
// kvengine/paged.py:197-205 and 288-311, with the values quantised on the way.
//
// The mathematics. A block whose first new row is its first row takes the scale of the
// largest new value (q8_scale). A block that holds rows of earlier passes keeps its scale
// where that is large enough, and else takes the larger one, and its rows' codes follow
// (q8_rescale): the scale never falls while a row is held, so a row is rounded again only
// when a later one outgrows its block. Values are rounded once to 8 bits, to the nearest.
//
// One wave per (sequence, touched block, kv head, K or V): it owns the block's tile, so the
// maximum, the scale and the codes need no other wave. The tile goes 16 tokens at a time:
// lane (lr, lg) reads CH = D / 16 channels of the tokens 4 lg .. 4 lg + 3, 16 lanes a row. K's
// codes lie as they were read; V's, channel-major, are turned in registers: 4 x 4 bytes by
// byte permutes (4 tokens of a channel in a word), then 4 x 4 words across the four lane groups
// by two lane swaps, so that a lane stores 16 tokens of a channel at once.
//
// What bounds it: one decode step is launch and three dependent reads (length, block id, scale
// and held codes): 32 sequences of 2 heads of 128 5.4 us. A prompt is bytes: 8 x 2049 tokens 9.0
// us, 2.8 TB/s; a tile's reads, its maximum and its stores follow one another in 4128 waves, four a
// SIMD (110 registers at head_dim 128), of which the last 32 find no place beside the rest (18 with a
// workgroup a tile, whose waves meet for the maximum and whose reads of V jump from token to token).

#include "kve_q8.h"

#include <type_traits>

namespace kve {

struct Q8WriteArgs {
  const void *k_new, *v_new;
  int64_t stride;  // elements between tokens
  uint8_t *k_pool, *v_pool;
  float *k_scale, *v_scale;  // [num_blocks][Hkv]
  const int32_t *tables, *seq_rows, *start_pos, *q_lens;
  int Tq, Hkv, D, bs, max_blocks, num_rows, num_blocks;
  int spans;      // blocks that Tq tokens can touch
  int64_t units;  // waves
};

constexpr int kWriteThreads = 256;

// 4 x 4 bytes: byte r of w[c] is byte c of q[r].
__device__ __forceinline__ void turn_bytes(const uint32_t (&q)[4], uint32_t* w) {
  const uint32_t a = __builtin_amdgcn_perm(q[1], q[0], 0x05010400u);
  const uint32_t b = __builtin_amdgcn_perm(q[3], q[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(q[1], q[0], 0x07030602u);
  const uint32_t d = __builtin_amdgcn_perm(q[3], q[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// 4 x 4 words across the lane groups: word r of group g is word g of group r.
__device__ __forceinline__ void turn_groups(uint32_t* w) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto x = __builtin_amdgcn_permlane32_swap(w[i], w[i + 2], false, false);
    w[i] = x[0];
    w[i + 2] = x[1];
  }
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const auto x = __builtin_amdgcn_permlane16_swap(w[i], w[i + 1], false, false);
    w[i] = x[0];
    w[i + 1] = x[1];
  }
}

// 0xff in the bytes of tokens [from, to) of the four that start at t
__device__ __forceinline__ uint32_t byte_mask(int t, int from, int to) {
  uint32_t m = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) m |= t + r >= from && t + r < to ? 0xffu << (8 * r) : 0u;
  return m;
}

template <typename E, Q8 Q, int D>
__global__ __launch_bounds__(kWriteThreads) void kv_write_q8_kernel(Q8WriteArgs a) {
  constexpr int CH = D / 16, NW = CH / 4;  // channels of a lane, words of their codes
  const int l = threadIdx.x & 63, lr = l & 15, lg = l >> 4;
  int64_t u64 = static_cast<int64_t>(blockIdx.x) * (kWriteThreads / 64) +
                __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (u64 >= a.units) return;
  int u = static_cast<int>(u64);
  const bool is_v = u & 1;
  u >>= 1;
  const int h = u % a.Hkv;
  u /= a.Hkv;
  const int i = u / a.spans, j = u - i * a.spans;
  const int T = a.q_lens ? min(a.q_lens[i], a.Tq) : a.Tq;
  const int row = a.seq_rows ? a.seq_rows[i] : i;
  if (T <= 0 || row < 0 || row >= a.num_rows) return;
  const int start = a.start_pos[row];
  if (start < 0 || start > INT32_MAX - a.bs - T) return;
  const int lb = start / a.bs + j;
  if (lb >= a.max_blocks) return;
  // the block's rows: [0, o) of earlier passes, [o, e) new, the others not in use
  const int base = lb * a.bs;
  const int o = max(start - base, 0), e = min(start + T - base, a.bs);
  if (e <= o) return;
  const int blk = a.tables[static_cast<size_t>(row) * a.max_blocks + lb];
  const E* src = static_cast<const E*>(is_v ? a.v_new : a.k_new) +
                 static_cast<int64_t>(i) * a.Tq * a.stride + static_cast<int64_t>(h) * D + lr * CH;
  const int first = base - start;  // the pass's token at the block's row 0

  // the lane's four tokens of the 16 that start at row t0 (zeros where they are not new)
  const auto read = [&](int t0, float (&x)[4][CH]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = t0 + 4 * lg + r;
      struct alignas(CH * sizeof(E) < 16 ? CH * sizeof(E) : 16) Vec { E v[CH]; };
      // (a row of the pass either way)
      const Vec v = *reinterpret_cast<const Vec*>(src + (first + min(max(t, o), e - 1)) * a.stride);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float y;
        if constexpr (std::is_same_v<E, float>) y = v.v[c];
        else y = bf16_to_f32(v.v[c]);
        x[r][c] = t >= o && t < e ? y : 0.0f;
      }
    }
  };
  const auto largest = [&](const float (&x)[4][CH], float m) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int c = 0; c < CH; ++c) m = fmaxf(m, fabsf(x[r][c]) < INFINITY ? fabsf(x[r][c]) : 0.0f);
    }
    return m;
  };
  // the first 16 tokens that hold new ones stay in registers: with blocks of 16, all
  const int t_first = o & ~15;
  float x[4][CH];
  read(t_first, x);
  if (blk < 0 || blk >= a.num_blocks) return;
  const size_t tile = static_cast<size_t>(blk) * a.Hkv + h;
  uint8_t* codes = (is_v ? a.v_pool : a.k_pool) + tile * a.bs * D;
  float* scale = (is_v ? a.v_scale : a.k_scale) + tile;
  const float s0 = o > 0 ? *scale : 0.0f;
  // V's codes beside the new ones, asked for with the scale
  const auto v_at = [&](int w, int t0) {  // channel lr CH + 4 w + lg, 16 tokens
    return reinterpret_cast<u32x4*>(codes + static_cast<size_t>(lr * CH + 4 * w + lg) * a.bs + t0);
  };
  u32x4 was[NW];
  if (is_v && (t_first < o || t_first + 16 > e)) {
#pragma unroll
    for (int w = 0; w < NW; ++w) was[w] = *v_at(w, t_first);
  }
  float m = largest(x, 0.0f);
  for (int t0 = t_first + 16; t0 < e; t0 += 16) {
    float y[4][CH];
    read(t0, y);
    m = largest(y, m);
  }
  m = fmaxf(m, dpp_mov<0xB1>(m));
  m = fmaxf(m, dpp_mov<0x4E>(m));
  m = fmaxf(m, dpp_mov<0x141>(m));
  m = fmaxf(m, dpp_mov<0x140>(m));
  m = max_across_groups(m);
  const float s = fmaxf(s0, q8_scale<Q>(m)), inv = q8_inv(s);
  const bool grown = s != s0;
  if (l == 0) *scale = s;
  for (int t0 = o > 0 && grown ? 0 : t_first; t0 < e; t0 += 16) {
    if (t0 > t_first) read(t0, x);
    uint32_t q[4][NW];  // [token][4 channels a word]
    if (t0 >= t_first) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = t0 + 4 * lg + r;
        // (a decode step's one row is one lane group's, and one of four turns)
        if (!__any(t >= o && t < e)) {
#pragma unroll
          for (int w = 0; w < NW; ++w) q[r][w] = 0;
          continue;
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float y[4] = {x[r][4 * w], x[r][4 * w + 1], x[r][4 * w + 2], x[r][4 * w + 3]};
          q[r][w] = q8_codes<Q>(y, s, inv);
        }
      }
    }
    if (!is_v) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = t0 + 4 * lg + r;
        uint32_t* at = reinterpret_cast<uint32_t*>(codes + static_cast<size_t>(t) * D + lr * CH);
        if (t < o && grown) {
#pragma unroll
          for (int w = 0; w < NW; ++w) at[w] = q8_rescale<Q>(at[w], s0, s);
        } else if (t >= o && t < e) {
          if constexpr (NW == 2) *reinterpret_cast<u32x2*>(at) = u32x2{q[r][0], q[r][1]};
          else at[0] = q[r][0];
        }
      }
      continue;
    }
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      u32x4 out = {0, 0, 0, 0};
      if (t0 >= t_first) {
        const uint32_t rows[4] = {q[0][w], q[1][w], q[2][w], q[3][w]};
        uint32_t turned[4];
        turn_bytes(rows, turned);
        turn_groups(turned);
        out = u32x4{turned[0], turned[1], turned[2], turned[3]};
      }
      if (t0 < o || t0 + 16 > e) {
        const u32x4 before = t0 == t_first ? was[w] : *v_at(w, t0);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t fresh = byte_mask(t0 + 4 * g, o, e), held = byte_mask(t0 + 4 * g, 0, o);
          uint32_t old = before[g];
          if (grown && o > 0) old = (q8_rescale<Q>(old, s0, s) & held) | (old & ~held);
          out[g] = (out[g] & fresh) | (old & ~fresh);
        }
      }
      *v_at(w, t0) = out;
    }
  }
}

template <typename E, Q8 Q>
static void launch_write_q8(const Q8WriteArgs& a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((a.units + 3) / 4));
  if (a.D == 64)
    hipLaunchKernelGGL((kv_write_q8_kernel<E, Q, 64>), grid, dim3(kWriteThreads), 0, st, a);
  else
    hipLaunchKernelGGL((kv_write_q8_kernel<E, Q, 128>), grid, dim3(kWriteThreads), 0, st, a);
}

template <typename E>
static void launch_write_q8(const Q8WriteArgs& a, int pool, hipStream_t st) {
  if (pool == KVE_DTYPE_I8) launch_write_q8<E, Q8::kInt8>(a, st);
  else launch_write_q8<E, Q8::kE4m3>(a, st);
}

}  // namespace kve

using namespace kve;

extern "C" int kve_kv_write_q8(const void* k_new, const void* v_new, int64_t src_token_stride,
                               void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                               const int32_t* block_tables, const int32_t* seq_rows,
                               const int32_t* start_pos, const int32_t* q_lens, int num_seqs,
                               int q_len, int num_kv_heads, int head_dim, int block_size,
                               int max_blocks, int num_rows, int num_blocks, int dtype,
                               int pool_dtype, void* stream) {
  clear_error();
  if (num_seqs == 0) return KVE_OK;
  KVE_REQUIRE(k_new && v_new && k_pool && v_pool && k_scale && v_scale && block_tables && start_pos,
              "kve_kv_write_q8: null pointer argument");
  KVE_REQUIRE(num_seqs > 0 && q_len > 0 && num_kv_heads > 0 && max_blocks > 0 && num_rows > 0 &&
                  num_blocks > 0,
              "kve_kv_write_q8: bad sizes");
  KVE_REQUIRE(block_size > 0 && block_size % 16 == 0 && block_size <= (1 << 20),
              "kve_kv_write_q8: block_size %d (a multiple of 16)", block_size);
  KVE_REQUIRE(dtype == KVE_DTYPE_BF16 || dtype == KVE_DTYPE_F32, "kve_kv_write_q8: dtype %d", dtype);
  KVE_REQUIRE(pool_dtype == KVE_DTYPE_I8 || pool_dtype == KVE_DTYPE_E4M3,
              "kve_kv_write_q8: pool dtype %d", pool_dtype);
  KVE_REQUIRE(head_dim == 64 || head_dim == 128, "kve_kv_write_q8: head_dim %d (64 or 128)", head_dim);
  const int vec = dtype == KVE_DTYPE_BF16 ? 8 : 4;
  KVE_REQUIRE(src_token_stride >= static_cast<int64_t>(num_kv_heads) * head_dim &&
                  src_token_stride % vec == 0,
              "kve_kv_write_q8: src_token_stride %lld", static_cast<long long>(src_token_stride));
  KVE_REQUIRE(((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new) |
                reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0,
              "kve_kv_write_q8: rows and pools must be 16-byte aligned");
  Q8WriteArgs a{};
  a.k_new = k_new;
  a.v_new = v_new;
  a.stride = src_token_stride;
  a.k_pool = static_cast<uint8_t*>(k_pool);
  a.v_pool = static_cast<uint8_t*>(v_pool);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.tables = block_tables;
  a.seq_rows = seq_rows;
  a.start_pos = start_pos;
  a.q_lens = q_lens;
  a.Tq = q_len;
  a.Hkv = num_kv_heads;
  a.D = head_dim;
  a.bs = block_size;
  a.max_blocks = max_blocks;
  a.num_rows = num_rows;
  a.num_blocks = num_blocks;
  // tokens o .. o + q_len - 1 of a block offset o <= block_size - 1
  a.spans = static_cast<int>((static_cast<int64_t>(q_len) + block_size - 2) / block_size) + 1;
  a.units = static_cast<int64_t>(num_seqs) * a.spans * num_kv_heads * 2;
  // (a launch has below 2^32 threads)
  KVE_REQUIRE(a.units < (1ll << 26), "kve_kv_write_q8: %d x %d tokens too large for one launch",
              num_seqs, q_len);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == KVE_DTYPE_BF16) launch_write_q8<uint16_t>(a, pool_dtype, st);
  else launch_write_q8<float>(a, pool_dtype, st);
  return check_launch("kve_kv_write_q8");
}
