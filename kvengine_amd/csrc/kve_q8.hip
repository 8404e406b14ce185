// New K/V rows into a cache held in 8 bits (kve_kv_write_q8): the paged scatter of
// kvengine/paged.py:197-205 and 288-311, with the values quantised on the way.
//
// The mathematics. A block whose first new row is its first row takes the scale of the
// largest new value (q8_scale). A block that holds rows of earlier passes keeps its scale
// where that is large enough, and else takes the larger one, and its rows' codes follow
// (q8_rescale): the scale never falls while a row is held, so a row is rounded again only
// when a later one outgrows its block. Values are rounded once to 8 bits, to the nearest.
//
// One workgroup per (sequence, touched block, kv head, K or V): it owns the block's tile,
// so the maximum, the scale and the codes need no other workgroup. A thread holds 8 values:
// of K 8 channels of a token, of V 8 tokens of a channel, which are 8 consecutive bytes of
// the tile either way.

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
  int spans;  // blocks that Tq tokens can touch
};

constexpr int kWriteThreads = 256;

template <typename E, Q8 Q>
__global__ __launch_bounds__(kWriteThreads) void kv_write_q8_kernel(Q8WriteArgs a) {
  __shared__ float sm_max[kWriteThreads / 64];
  const int tid = threadIdx.x;
  const bool is_v = blockIdx.x & 1;
  int u = blockIdx.x >> 1;
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
  if (blk < 0 || blk >= a.num_blocks) return;
  const size_t tile = static_cast<size_t>(blk) * a.Hkv + h;
  uint8_t* codes = (is_v ? a.v_pool : a.k_pool) + tile * a.bs * a.D;
  float* scale = (is_v ? a.v_scale : a.k_scale) + tile;
  const float s0 = o > 0 ? *scale : 0.0f;
  const E* src = static_cast<const E*>(is_v ? a.v_new : a.k_new) +
                 static_cast<int64_t>(i) * a.Tq * a.stride + static_cast<int64_t>(h) * a.D;
  const int first = base - start;  // the pass's token at the block's row 0

  const auto to_float = [](E v) {
    if constexpr (std::is_same_v<E, float>) return v;
    else return bf16_to_f32(v);
  };
  // Item n of the tile: 8 values, (token, channel) of its value c
  const int items = a.bs * a.D / 8;
  const auto read = [&](int n, float (&x)[8]) {
    if (is_v) {
      const int ch = n % a.D, t0 = n / a.D * 8;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        x[c] = t0 + c >= o && t0 + c < e ? to_float(src[(first + t0 + c) * a.stride + ch]) : 0.0f;
    } else {
      const int t = n * 8 / a.D, d0 = n * 8 % a.D;
      if (t >= o && t < e) {
        const E* p = src + (first + t) * a.stride + d0;
        struct alignas(16) Vec { E v[16 / sizeof(E)]; };
#pragma unroll
        for (int w = 0; w < 8; w += 16 / sizeof(E)) {
          const Vec vec = *reinterpret_cast<const Vec*>(p + w);
#pragma unroll
          for (int c = 0; c < static_cast<int>(16 / sizeof(E)); ++c) x[w + c] = to_float(vec.v[c]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = 0.0f;
      }
    }
  };
  float m = 0.0f;
  for (int n = tid; n < items; n += kWriteThreads) {
    float x[8];
    read(n, x);
#pragma unroll
    for (int c = 0; c < 8; ++c) m = fmaxf(m, fabsf(x[c]) < INFINITY ? fabsf(x[c]) : 0.0f);
  }
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) m = fmaxf(m, __shfl_xor(m, w));
  if ((tid & 63) == 0) sm_max[tid >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWriteThreads / 64; ++w) m = fmaxf(m, sm_max[w]);
  const float s = fmaxf(s0, q8_scale<Q>(m)), inv = q8_inv(s);
  if (tid == 0) *scale = s;
  const bool grown = s != s0;
  for (int n = tid; n < items; n += kWriteThreads) {
    // of the item's 8 rows (K: one row): which are new, which held
    const int t0 = is_v ? n / a.D * 8 : n * 8 / a.D, t1 = is_v ? t0 + 8 : t0 + 1;
    const bool some_new = t0 < e && t1 > o, some_old = t0 < o;
    if (!some_new && !(some_old && grown)) continue;
    uint2* at = reinterpret_cast<uint2*>(codes + (is_v ? static_cast<size_t>(n % a.D) * a.bs + t0
                                                       : static_cast<size_t>(n) * 8));
    float x[8];
    read(n, x);
    const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
    uint32_t w[2] = {q8_codes<Q>(lo, s, inv), q8_codes<Q>(hi, s, inv)};
    if (some_old || t1 > e) {
      const uint2 was = *at;
      const uint32_t old[2] = {grown && some_old ? q8_rescale<Q>(was.x, s0, s) : was.x,
                               grown && some_old ? q8_rescale<Q>(was.y, s0, s) : was.y};
      const uint32_t raw[2] = {was.x, was.y};
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int t = is_v ? t0 + c : t0;
        const uint32_t mask = 0xffu << (8 * (c & 3));
        if (t < o) w[c >> 2] = (w[c >> 2] & ~mask) | (old[c >> 2] & mask);
        else if (t >= e) w[c >> 2] = (w[c >> 2] & ~mask) | (raw[c >> 2] & mask);
      }
    }
    *at = uint2{w[0], w[1]};
  }
}

template <typename E>
static void launch_write_q8(const Q8WriteArgs& a, int pool, int grid, hipStream_t st) {
  if (pool == KVE_DTYPE_I8)
    hipLaunchKernelGGL((kv_write_q8_kernel<E, Q8::kInt8>), dim3(grid), dim3(kWriteThreads), 0, st, a);
  else
    hipLaunchKernelGGL((kv_write_q8_kernel<E, Q8::kE4m3>), dim3(grid), dim3(kWriteThreads), 0, st, a);
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
  KVE_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 1024, "kve_kv_write_q8: head_dim %d",
              head_dim);
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
  const int64_t grid = static_cast<int64_t>(num_seqs) * a.spans * num_kv_heads * 2;
  KVE_REQUIRE(grid < (1ll << 31), "kve_kv_write_q8: %d x %d tokens too large for one launch",
              num_seqs, q_len);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == KVE_DTYPE_BF16)
    launch_write_q8<uint16_t>(a, pool_dtype, static_cast<int>(grid), st);
  else
    launch_write_q8<float>(a, pool_dtype, static_cast<int>(grid), st);
  return check_launch("kve_kv_write_q8");
}
