// What the kernels of tree attention share: the step's arrays, a packed row's node and head, and what a node may look at.
//
// A step brings, per sequence, `q_len` nodes of a drafted tree behind `past = kv_len - q_len` cached tokens.  Node i's key and value
// are filed at place past + i of the sequence, whatever its position; its position (tok_pos, past + its depth) is what its
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
  const uint32_t* mask;      // [tokens, words]
  int words;
  int heads, kv_heads, dim;
  float scale_log2;          // scale * log2(e): exponentials are powers of two
  int window;                // 0: none
  int splits;                // parts a sequence's keys are cut into
  float* part_acc;           // [tokens, heads, splits, dim], parts that meet in the second kernel
  float* part_ml;            // [tokens, heads, splits, 2]: reference and sum
};

// Whether a node at `pos` whose mask stands at `bits` sees place j.
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, const uint32_t* bits, int pos, int past, int kv_len, const int* node_pos, int j) {
  if (j < past) return a.window == 0 || j > pos - a.window;
  const int m = j - past;
  if (j >= kv_len || m >= 32 * a.words || !((bits[m >> 5] >> (m & 31)) & 1u)) return false;
  return a.window == 0 || node_pos[m] > pos - a.window;
}

// Joins the parts of a (node, head): o = sum_s w_s acc_s / sum_s w_s l_s with w_s = 2^(m_s - max m).  A warp takes a
// head of a node; up to 32 parts.
template <typename T>
static __global__ void attention_tree_join_kernel(const TreeArgs a) {
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.y, node = blockIdx.x;
  if (node >= a.seq_q_len[seq]) return;
  const int lane = threadIdx.x & 31;
  const float* part_ml = a.part_ml;
  const float* part_acc = a.part_acc;
  SB_BEHIND_WAIT(part_ml);
  SB_BEHIND_WAIT(part_acc);
  const int h = blockIdx.z * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (h >= a.heads) return;
  const size_t at = (size_t)(a.seq_q_start[seq] + node) * a.heads + h, p0 = at * a.splits;
  // (up to 32 parts: one a lane)
  const float2 ml = lane < a.splits ? reinterpret_cast<const float2*>(part_ml)[p0 + lane] : make_float2(-INFINITY, 0.f);
  const float top = warp_max(ml.y != 0.f ? ml.x : -INFINITY);
  const float w = ml.y != 0.f ? exp2f(ml.x - top) : 0.f, sum = warp_sum(ml.y != 0.f ? ml.y * w : 0.f);
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  for (int d0 = 0; d0 < a.dim; d0 += 32) {
    const int d = d0 + lane;
    float o = 0.f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
      const float x = d < a.dim ? part_acc[(p0 + s) * a.dim + d] : 0.f, f = __shfl_sync(0xffffffffu, w, s);
      o = f != 0.f ? fmaf(x, f, o) : o;
    }
    if (d < a.dim) ((T*)a.out)[at * a.dim + d] = from_f<T>(o * inv);
  }
}
