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

struct TreeAcceptArgs {
  const int32_t *tokens, *parents, *preds, *node_counts, *lens, *seq_rows, *tables;
  int32_t *n_acc, *emitted, *path, *keep;
  void *k, *v;
  int num_rows, nodes, L, Hkv, D, bs, max_blocks, num_blocks;
};

// Grid (sequences, parts): every wave walks the sequence's tree (a few shuffles and
// ballots on values that one load each brought in), the first workgroup of a
// sequence writes the results, and all of them share the moves, a thread owning one
// 16-byte piece of a K row or one channel of V in one (layer, kv head) and taking
// the path's nodes in order. A node moves to a slot at or below its own and every
// later node lies above that slot, so a thread that reads kMoves nodes and then
// writes them never overwrites a node still to be read. K rows are contiguous; V is
// channel-major, so a moved token is one element of a 32-byte run per channel.
constexpr int kAcceptThreads = 256;
constexpr int kMoves = 8;

template <typename E>
__global__ __launch_bounds__(kAcceptThreads) void tree_accept_kernel(TreeAcceptArgs a) {
  const int i = blockIdx.x, l = threadIdx.x & 63;
  const int n = a.node_counts ? min(a.node_counts[i], a.nodes) : a.nodes;
  const int row = a.seq_rows ? a.seq_rows[i] : i;
  const bool has_row = a.lens && row >= 0 && row < a.num_rows;
  const int start = has_row ? a.lens[row] - max(n, 0) : 0;
  const size_t at = static_cast<size_t>(i) * a.nodes + l;
  const bool in = l < n;
  const int parent = tree_parent(a.parents + static_cast<size_t>(i) * a.nodes, l, n);
  const int token = in ? a.tokens[at] : 0, pred = in ? a.preds[at] : 0;

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

  if (!a.k || !has_row || start < 0) return;
  // nodes below the first gap in the path are where they belong
  if ((taken & (taken + 1)) == 0) return;
  const int j0 = __builtin_ctzll(~taken);
  if (a.seq_rows) {
    // two entries of one row would move its slots at once: the first one does
    bool again = false;
    for (int e = l; e < i; e += 64) again |= a.seq_rows[e] == row;
    if (__any(again)) return;
  }
  constexpr int VEC = 16 / sizeof(E);
  const int kpieces = a.D / VEC, per_head = kpieces + a.D;
  const int items = a.L * a.Hkv * per_head;
  const int32_t* table = a.tables + static_cast<size_t>(row) * a.max_blocks;
  const int cap = a.max_blocks * a.bs;
  for (int it = blockIdx.y * kAcceptThreads + threadIdx.x; it < items;
       it += gridDim.y * kAcceptThreads) {
    const int lh = it / per_head, c = it - lh * per_head;
    const int layer = lh / a.Hkv, h = lh - layer * a.Hkv;
    // element of (block, offset): a K piece c < kpieces, or V channel c - kpieces
    const size_t head0 = (static_cast<size_t>(layer) * a.num_blocks * a.Hkv + h) * a.bs * a.D;
    const size_t blk_step = static_cast<size_t>(a.Hkv) * a.bs * a.D;
    const bool is_k = c < kpieces;
    const int off_step = is_k ? a.D : 1;
    const size_t first = head0 + (is_k ? c * VEC : static_cast<size_t>(c - kpieces) * a.bs);
    uint64_t left = taken >> j0 << j0;
    int j = j0;
    while (left) {
      E* dst[kMoves];
      u32x4 kx[kMoves];
      E vx[kMoves];
      int m = 0;
#pragma unroll
      for (int q = 0; q < kMoves; ++q) {
        dst[q] = nullptr;
        if (!left) continue;
        const int node = __builtin_ctzll(left);
        left &= left - 1;
        const int sp = start + node, dp = start + j + m;
        ++m;
        if (sp >= cap) continue;
        const int sb = table[sp / a.bs], db = table[dp / a.bs];
        if (sb < 0 || sb >= a.num_blocks || db < 0 || db >= a.num_blocks) continue;
        const size_t so = first + sb * blk_step + static_cast<size_t>(sp % a.bs) * off_step;
        const size_t dof = first + db * blk_step + static_cast<size_t>(dp % a.bs) * off_step;
        dst[q] = static_cast<E*>(is_k ? a.k : a.v) + dof;
        if (is_k) kx[q] = *reinterpret_cast<const u32x4*>(static_cast<const E*>(a.k) + so);
        else vx[q] = static_cast<const E*>(a.v)[so];
      }
      j += m;
#pragma unroll
      for (int q = 0; q < kMoves; ++q) {
        if (!dst[q]) continue;
        if (is_k) *reinterpret_cast<u32x4*>(dst[q]) = kx[q];
        else *dst[q] = vx[q];
      }
    }
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
  int parts = 1;
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
    const long long items =
        static_cast<long long>(num_layers) * num_kv_heads * (head_dim / vec + head_dim);
    KVE_REQUIRE(items < (1ll << 30) && static_cast<long long>(max_blocks) * block_size < (1ll << 30),
                "kve_tree_accept: %d layers x %d heads, %d blocks a row: too large", num_layers,
                num_kv_heads, max_blocks);
    parts = static_cast<int>((items + kAcceptThreads - 1) / kAcceptThreads);
    if (parts > 1024) parts = 1024;
  }
  const TreeAcceptArgs a{tokens, parents, preds, node_counts, lens, seq_rows, block_tables,
                         n_acc, emitted, path, keep_lens, k_pool, v_pool, num_rows, nodes,
                         num_layers, num_kv_heads, head_dim, block_size, max_blocks, num_blocks};
  const dim3 grid(num_seqs, parts);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (k_pool && dtype == KVE_DTYPE_F32)
    hipLaunchKernelGGL(tree_accept_kernel<float>, grid, dim3(kAcceptThreads), 0, st, a);
  else
    hipLaunchKernelGGL(tree_accept_kernel<uint16_t>, grid, dim3(kAcceptThreads), 0, st, a);
  return check_launch("kve_tree_accept");
}
