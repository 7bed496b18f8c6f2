// What the kernels of tree attention share: the step's arrays, a packed row's node and head, and what a node may look at.
//
// A step brings, per sequence, `q_len` nodes of a drafted tree behind `past = kv_len - q_len` cached tokens.  Node i's key and value
// are filed at place past + i of the sequence, whatever its position; its position (tok_pos, past + its depth, below kv_len) is what its
// rotation and a window go by.  With mask_i the bits of the nodes that node i looks at (itself and those above it, or what the caller
// likes):
//     o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i k_j),
// over the places j < past (in a window w: j > pos_i - w) and j = past + m with bit m of mask_i set (in a window: pos_m > pos_i - w).
// A node that sees nothing gets zeros.  The query heads of a key/value head read the same keys, so a tile's rows are the (node, head)
// pairs of one key/value head, node by node: packed row r is head r % group of node r / group.
#pragma once

#include "common.cuh"

struct TreeArgs {
  const void* q;             // [tokens, heads * dim]
  void* out;                 // the same
  const void* k_store;       // [pages, kv_heads, 64, dim]
  const void* v_store;
  const int* block_table;    // [slots, table_stride]
  int table_stride;
  const int* seq_slot;       // per sequence: its slot, its first row, its rows, its length with them
  const int* seq_q_start;
  const int* seq_q_len;
  const int* seq_kv_len;
  const int* tok_pos;        // [tokens]
  const uint32_t* mask;      // [tokens, mask_stride]
  int mask_stride, words;    // words a row holds; those of them that nodes can have (at most TREE_MAX_WORDS)
  int heads, kv_heads, dim;
  float scale_log2;          // scale * log2(e): exponentials are powers of two
  int window;                // 0: none
  int splits;                // parts a sequence's keys are cut into: the blocks of a cluster
};

// The end of a cluster whose blocks have read from one another: nobody leaves before all have what they read.  (Relaxed: what a thread read it has used
// by now, and a release would wait for its results' way to memory.)
__device__ __forceinline__ void tree_cluster_leave() {
  __syncwarp();                            // (.aligned: a whole warp at once)
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

#define TREE_MAX_WORDS 8                  // of a mask: 256 nodes

// Which of the places j0 .. j0 + 63 a row sees, as bits: bits[] is its mask (TREE_MAX_WORDS words, without the nodes in front of its window),
// `first` its window's first place (0: no window).
__device__ __forceinline__ uint64_t tree_view(const uint32_t* bits, int first, int past, int kv_len, int j0) {
  uint64_t view = 0;
  const int m0 = j0 - past;                 // the first place's node, or minus how many cached places come first
  if (m0 > -64) {
    const int w = max(m0, 0) >> 5, shift = max(m0, 0) & 31;
    uint64_t nodes = 0;
    if (w < TREE_MAX_WORDS) {
      nodes = (uint64_t)bits[w] | (uint64_t)(w + 1 < TREE_MAX_WORDS ? bits[w + 1] : 0u) << 32;
      if (shift) nodes = nodes >> shift | (uint64_t)(w + 2 < TREE_MAX_WORDS ? bits[w + 2] : 0u) << (64 - shift);
    }
    view = m0 < 0 ? nodes << -m0 | ((1ull << -m0) - 1) : nodes;
  } else {
    view = ~0ull;
  }
  const int end = kv_len - j0, hidden = min(first, past) - j0;
  if (end < 64) view &= end > 0 ? (1ull << end) - 1 : 0ull;          // places behind the sequence
  if (hidden > 0) view &= hidden < 64 ? ~0ull << hidden : 0ull;      // cached places in front of the window
  return view;
}
// The first place any node sees and the one from which on every node sees all that is cached, as far as the lengths say: positions lie between the first
// behind what is cached and the sequence's last, so nothing has to be read for them.
__device__ __forceinline__ int tree_low(const TreeArgs& a, int past) { return a.window > 0 ? max(past - a.window + 1, 0) : 0; }
__device__ __forceinline__ int tree_high(const TreeArgs& a, int past, int kv_len) { return a.window > 0 ? min(max(kv_len - a.window, 0), past) : 0; }
// Word w of the mask of a sequence's node, without the nodes in front of its window (first: its first place; up to `past` it leaves out none).
__device__ __forceinline__ uint32_t tree_mask_word(const TreeArgs& a, int start, int node, int w, int q_len, int first, int past) {
  uint32_t bits = w < a.words ? a.mask[(size_t)(start + node) * a.mask_stride + w] : 0u;
  if (a.window > 0 && first > past) {
    for (uint32_t left = bits; left; left &= left - 1) {
      const int m = 32 * w + __ffs(left) - 1;
      if (m >= q_len || a.tok_pos[start + m] < first) bits &= ~(left & -left);
    }
  }
  return bits;
}
