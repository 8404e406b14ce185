// Trees of drafted tokens: the masks and depths that a tree's attention and rotary
// positions take, and the accept that walks the tree and moves the accepted path's
// K/V to consecutive slots. The attention itself is verify_attn_*_kernel<TREE>
// (kve_attn.hip). No counterpart in the reference, whose drafts are chains
// (kvengine/speculative.py:111-215).
//
// A tree has at most 64 nodes, so one wave holds it, a node per lane, and a set of
// nodes is one 64-bit mask. Parents stand before their children, so along any path
// the node numbers grow: the set bits of an accepted path's mask, lowest first, are
// the path.

#include "kve_common.h"

#include <type_traits>

namespace kve {

// The parent of lane t's node, or -1: none, or no node before t.
__device__ __forceinline__ int tree_parent(const int32_t* parents, int t, int n) {
  const int p = t < n ? parents[t] : -1;
  return p < t ? p : -1;  // (a negative one below -1 is read as none by its sign)
}

// One wave per sequence. Pointer doubling: after r rounds a lane's mask holds its
// nearest 2^r nodes (itself included) and p its 2^r-th ancestor, so six rounds
// cover 64 nodes. Launch bound: 32 x 64 nodes are 24 KB of results.
__global__ __launch_bounds__(64) void tree_masks_kernel(const int32_t* parents,
                                                        const int32_t* node_counts, int nodes,
                                                        int64_t* masks, int32_t* depths) {
  const int i = blockIdx.x, t = threadIdx.x;
  const int n = node_counts ? min(node_counts[i], nodes) : nodes;
  int p = tree_parent(parents + static_cast<size_t>(i) * nodes, t, n);
  uint32_t lo = t < 32 ? 1u << t : 0u, hi = t < 32 ? 0u : 1u << (t - 32);
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    const int from = p < 0 ? t : p;
    const uint32_t plo = __shfl(lo, from), phi = __shfl(hi, from);
    const int pp = __shfl(p, from);
    if (p >= 0) {
      lo |= plo;
      hi |= phi;
      p = pp;
    }
  }
  if (t >= nodes) return;
  const bool live = t < n;
  const size_t at = static_cast<size_t>(i) * nodes + t;
  if (masks) masks[at] = live ? static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo) : 0;
  if (depths) depths[at] = live ? __popc(lo) + __popc(hi) - 1 : 0;
}

// n / d for 0 <= n < 2^30 without the divide's thirty instructions: with 2^(s-1) < d <=
// 2^s, mul = ceil(2^(30+s) / d) is too large by less than one, so that n mul / 2^(30+s)
// passes n / d by less than 2^30 / 2^(30+s) <= 1 / d, too little to reach the next whole.
struct Divisor {
  uint32_t mul, shift;
  explicit Divisor(int d) {
    uint32_t s = 0;
    while ((1ll << s) < d) ++s;
    shift = 30 + s;
    mul = static_cast<uint32_t>(((1ull << shift) + d - 1) / d);
  }
  __device__ int operator()(int n) const {
    return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul >> shift);
  }
};

struct TreeAcceptArgs {
  const int32_t *tokens, *parents, *preds, *node_counts, *lens, *seq_rows, *tables;
  int32_t *n_acc, *emitted, *path, *keep;
  void *k, *v;
  int num_rows, nodes, L, Hkv, D, bs, max_blocks, num_blocks;
  Divisor by_kwidth, by_dim, by_kv;  // K's pieces a row, head_dim, the kv heads
};

// Grid (sequences, parts): every wave walks the sequence's tree (a few shuffles and
// ballots on values that one load each brought in), the first workgroup of a
// sequence writes the results, and all of them share the moves. What bounds it is the
// way to the data: the launch and the tree's loads 4 us, then K/V that nothing has
// touched since the forward, pages apart from layer to layer: 32 trees of 16 nodes in 36
// layers of 2 heads of 128 move 3.1 MB in 14.6 us (21.0 with a lane taking all of its
// column's moves, whose loads under branches waited for each other).
constexpr int kAcceptThreads = 256;
constexpr int kMoves = 8;  // loads in flight of a lane

// Where a lane's move takes from and puts to: element offsets in a layer's first head.
struct Move {
  size_t from, to;
  bool live;
};

// The moves of 64 columns of one pool, `columns` in all and `width` a kv head: K's
// pieces of 16 bytes or V's channels, T one of either, column c of a slot at c * cstep.
// 2^lg lanes share a column, a move each, so that all of a column's loads are one
// instruction and come before its stores, whichever slots they overlap; the 2^lg turns
// that the wave takes for its 64 columns are loaded Q at a time. Every lane loads (one
// with nothing to move loads its column's slot 0 of block 0): a load under a branch is
// waited for before the next.
template <int Q, typename T>
__device__ __forceinline__ void move_columns(T* pool, size_t layer_stride, size_t head_stride,
                                             int first, int columns, int width, Divisor by_width,
                                             int Hkv, Divisor by_kv, int cstep, Move mv, int lg) {
  const int l = threadIdx.x & 63;
  for (int turn = 0; turn < 1 << lg; turn += Q) {
    T *dst[Q], x[Q];
    bool ok[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int column = first + (turn + q) * (64 >> lg) + (l >> lg);
      ok[q] = mv.live && column < columns;
      const int at = min(column, columns - 1), lh = by_width(at), layer = by_kv(lh);
      T* base = pool + layer * layer_stride + (lh - layer * Hkv) * head_stride +
                (at - lh * width) * cstep;
      x[q] = base[mv.from];
      dst[q] = base + mv.to;
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) asm volatile("" ::"v"(x[q]));  // (or it loads under `ok`)
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (ok[q]) *dst[q] = x[q];
  }
}

template <typename T>
__device__ __forceinline__ void move_columns(T* pool, size_t layer_stride, size_t head_stride,
                                             int first, int columns, int width, Divisor by_width,
                                             int Hkv, Divisor by_kv, int cstep, Move mv, int lg) {
  const auto go = [&](auto q) {
    move_columns<decltype(q)::value>(pool, layer_stride, head_stride, first, columns, width,
                                     by_width, Hkv, by_kv, cstep, mv, lg);
  };
  if (lg >= 3) go(std::integral_constant<int, kMoves>{});
  else if (lg == 2) go(std::integral_constant<int, 4>{});
  else if (lg == 1) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 1>{});
}

template <typename E>
__global__ __launch_bounds__(kAcceptThreads) void tree_accept_kernel(TreeAcceptArgs a) {
  const int i = blockIdx.x, l = threadIdx.x & 63;
  const int n = a.node_counts ? min(a.node_counts[i], a.nodes) : a.nodes;
  const int row = a.seq_rows ? a.seq_rows[i] : i;
  const bool has_row = a.lens && row >= 0 && row < a.num_rows;
  const int start = has_row ? a.lens[row] - max(n, 0) : 0;
  // all loads before the walk: one wait instead of one after the other
  const size_t at = static_cast<size_t>(i) * a.nodes + l;
  int parent = -1, token = 0, pred = 0;
  if (l < a.nodes) {
    parent = a.parents[at];
    token = a.tokens[at];
    pred = a.preds[at];
  }
  // lane t: slot start + t, as its block (-1: none) and its offset in it
  const bool moving = a.k && has_row && start >= 0;
  int blk = -1, off = 0;
  if (moving) {
    const uint32_t slot = static_cast<uint32_t>(start) + l, entry = slot / a.bs;
    off = slot - entry * a.bs;
    if (entry < static_cast<uint32_t>(a.max_blocks))
      blk = a.tables[static_cast<size_t>(row) * a.max_blocks + entry];
    if (blk >= a.num_blocks) blk = -1;
  }
  const bool in = l < n;
  if (!in || parent >= l) parent = -1;

  uint64_t taken = n > 0 ? 1 : 0;
  int cur = 0;
  while (n > 0) {  // every turn moves to a higher node
    const int want = __builtin_amdgcn_readlane(pred, cur);
    const uint64_t kids = __ballot(in && parent == cur && token == want);
    if (!kids) break;
    cur = __builtin_ctzll(kids);
    taken |= 1ull << cur;
  }
  const int steps = __popcll(taken);  // nodes walked, node 0 included
  const int last = __builtin_amdgcn_readlane(pred, cur);

  if (blockIdx.y == 0 && threadIdx.x < 64) {
    if (l < a.nodes) {
      if (l >= steps) {
        a.path[at] = -1;
        a.emitted[at] = -1;
      } else if (l == steps - 1) {
        a.emitted[at] = last;
      }
    }
    if (taken >> l & 1) {
      const int j = __popcll(taken & ((1ull << l) - 1));
      int32_t* base = a.path + static_cast<size_t>(i) * a.nodes;
      base[j] = l;
      if (j > 0) a.emitted[static_cast<size_t>(i) * a.nodes + j - 1] = token;
    }
    if (l == 0) {
      a.n_acc[i] = max(steps - 1, 0);
      if (a.keep) a.keep[i] = has_row ? start + steps : 0;
    }
  }

  if (!moving) return;
  // nodes below the first gap in the path are where they belong
  if ((taken & (taken + 1)) == 0) return;
  const int j0 = __builtin_ctzll(~taken);
  if (a.seq_rows) {
    // two entries of one row would move its slots at once: the first one does
    bool again = false;
    for (int e = l; e < i; e += 64) again |= a.seq_rows[e] == row;
    if (__any(again)) return;
  }
  // P lanes to a column, P the power of two that holds the moves; lane l takes move
  // l mod P: the node that becomes the path's entry j0 + l mod P
  const int moves = steps - j0, lg = moves > 1 ? 32 - __builtin_clz(moves - 1) : 0;
  const int move = l & ((1 << lg) - 1), to = min(j0 + move, 63);
  // (lanes off the path write to the last entry, which then is not the path's)
  const int entry_of = taken >> l & 1 ? __popcll(taken & ((1ull << l) - 1)) : 63;
  const int from = __shfl(__builtin_amdgcn_ds_permute(4 * entry_of, l), to) & 63;
  const int sb = __shfl(blk, from), so = __shfl(off, from);
  const int db = __shfl(blk, to), dof = __shfl(off, to);
  const bool live = move < moves && sb >= 0 && db >= 0;
  const auto mv = [&](size_t head, int step) {
    return live ? Move{sb * (a.Hkv * head) + so * step, db * (a.Hkv * head) + dof * step, true}
                : Move{0, 0, false};
  };

  const int kw = a.D / static_cast<int>(16 / sizeof(E)), heads = a.L * a.Hkv;
  const int kchunks = cdiv(heads * kw, 64), chunks = kchunks + cdiv(heads * a.D, 64);
  const size_t khead = static_cast<size_t>(a.bs) * kw, vhead = static_cast<size_t>(a.bs) * a.D;
  const Move mk = mv(khead, kw), mvv = mv(vhead, 1);
  // a wave's 64 columns lie together: it meets one head's pages or two's
  for (int c = blockIdx.y * (kAcceptThreads / 64) + (threadIdx.x >> 6); c < chunks;
       c += gridDim.y * (kAcceptThreads / 64)) {
    if (c < kchunks)
      move_columns(static_cast<u32x4*>(a.k), a.num_blocks * (a.Hkv * khead), khead, c * 64,
                   heads * kw, kw, a.by_kwidth, a.Hkv, a.by_kv, 1, mk, lg);
    else
      move_columns(static_cast<E*>(a.v), a.num_blocks * (a.Hkv * vhead), vhead,
                   (c - kchunks) * 64, heads * a.D, a.D, a.by_dim, a.Hkv, a.by_kv, a.bs, mvv, lg);
  }
}

}  // namespace kve

using namespace kve;

extern "C" int kve_tree_masks(const int32_t* parents, const int32_t* node_counts, int num_seqs,
                              int nodes, int64_t* masks, int32_t* depths, void* stream) {
  clear_error();
  if (num_seqs == 0) return KVE_OK;
  KVE_REQUIRE(parents && (masks || depths), "kve_tree_masks: null pointer argument");
  KVE_REQUIRE(num_seqs > 0 && nodes > 0 && nodes <= KVE_TREE_MAX_NODES,
              "kve_tree_masks: %d sequences of %d nodes (at most %d)", num_seqs, nodes,
              KVE_TREE_MAX_NODES);
  hipLaunchKernelGGL(tree_masks_kernel, dim3(num_seqs), dim3(64), 0,
                     static_cast<hipStream_t>(stream), parents, node_counts, nodes, masks, depths);
  return check_launch("kve_tree_masks");
}

extern "C" int kve_tree_accept(const int32_t* tokens, const int32_t* parents, const int32_t* preds,
                               const int32_t* node_counts, const int32_t* lens, int num_rows,
                               const int32_t* seq_rows, int num_seqs, int nodes, int32_t* n_acc,
                               int32_t* emitted, int32_t* path, int32_t* keep_lens, void* k_pool,
                               void* v_pool, const int32_t* block_tables, int num_layers,
                               int num_kv_heads, int head_dim, int block_size, int max_blocks,
                               int num_blocks, int dtype, void* stream) {
  clear_error();
  if (num_seqs == 0) return KVE_OK;
  KVE_REQUIRE(tokens && parents && preds && n_acc && emitted && path,
              "kve_tree_accept: null pointer argument");
  KVE_REQUIRE(num_seqs > 0 && nodes > 0 && nodes <= KVE_TREE_MAX_NODES,
              "kve_tree_accept: %d sequences of %d nodes (at most %d)", num_seqs, nodes,
              KVE_TREE_MAX_NODES);
  KVE_REQUIRE(!(k_pool || keep_lens) || (lens && num_rows > 0),
              "kve_tree_accept: the pools and keep_lens need lens");
  KVE_REQUIRE(!k_pool == !v_pool, "kve_tree_accept: k_pool and v_pool go together");
  int parts = 1, kwidth = 1;
  if (k_pool) {
    KVE_REQUIRE(block_tables && num_layers > 0 && num_kv_heads > 0 && block_size > 0 &&
                    max_blocks > 0 && num_blocks > 0,
                "kve_tree_accept: bad sizes");
    KVE_REQUIRE(dtype == KVE_DTYPE_BF16 || dtype == KVE_DTYPE_F32, "kve_tree_accept: dtype %d",
                dtype);
    const int vec = dtype == KVE_DTYPE_BF16 ? 8 : 4;
    KVE_REQUIRE(head_dim > 0 && head_dim % vec == 0, "kve_tree_accept: head_dim %d", head_dim);
    KVE_REQUIRE(((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0,
                "kve_tree_accept: k_pool and v_pool must be 16-byte aligned");
    kwidth = head_dim / vec;
    const long long items =
        static_cast<long long>(num_layers) * num_kv_heads * (kwidth + head_dim);
    KVE_REQUIRE(items < (1ll << 30) && static_cast<long long>(max_blocks) * block_size < (1ll << 30),
                "kve_tree_accept: %d layers x %d heads, %d blocks a row: too large", num_layers,
                num_kv_heads, max_blocks);
    parts = static_cast<int>(items / kAcceptThreads + 1);
    if (parts > 1024) parts = 1024;
  }
  const TreeAcceptArgs a{tokens, parents, preds, node_counts, lens, seq_rows, block_tables,
                         n_acc, emitted, path, keep_lens, k_pool, v_pool, num_rows, nodes,
                         num_layers, num_kv_heads, head_dim, block_size, max_blocks, num_blocks,
                         Divisor(kwidth), Divisor(k_pool ? head_dim : 1),
                         Divisor(k_pool ? num_kv_heads : 1)};
  const dim3 grid(num_seqs, parts);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (k_pool && dtype == KVE_DTYPE_F32)
    hipLaunchKernelGGL(tree_accept_kernel<float>, grid, dim3(kAcceptThreads), 0, st, a);
  else
    hipLaunchKernelGGL(tree_accept_kernel<uint16_t>, grid, dim3(kAcceptThreads), 0, st, a);
  return check_launch("kve_tree_accept");
}
