// What a cache does with its pages beside attention: the rows of accepted drafts moved together, and whole pages copied.
#include "common.cuh"

// ------------------------------------------------------------------------------------------ accepted drafts
//
// A step has run the nodes of a drafted tree (attention_tree.cuh) and drawn a token behind every one of them.  The walk starts at the
// root (a sequence's first node) and goes on to a child whose token is the one that was drawn at its parent, the lowest of them, until
// there is none: exactly the tokens that one-token steps would have drawn.  Node c's parent is parents[c] (its place among the
// sequence's nodes, below c; anything else: c is nobody's child).  The nodes on the way lie at places past + path[i] of the
// sequence; they belong at past + i, and their keys and values go there.
//
// Every block walks its sequence's tree itself (a few shared-memory steps of a tree's depth; as a launch of its own it would cost more),
// then moves a 128-byte column of the keys or values of some (entry, key/value head) pairs: all rows are read to shared memory before
// any is written, so rows may overlap in any way.
#define CA_THREADS 128
#define CA_COLUMN 128                    // bytes of a row a block moves
#define CA_MAX_NODES 256

struct AcceptArgs {
  uint8_t* store[2];                     // keys, values: [entries, pages, kv_heads, 64, row_bytes]
  int row_bytes[2];
  long long entry_rows;                  // rows (of row_bytes) between entries: pages * kv_heads * 64
  int pairs, kv_heads;                   // entries * kv_heads
  const int* block_table;
  int table_stride;
  const int* seq_slot;
  const int* seq_q_start;
  const int* seq_q_len;
  const int* seq_kv_len;
  const int* tokens;                     // [rows]: the nodes' tokens, parents and what was drawn behind them
  const int* parents;
  const int* drawn;
  int* count;                            // [seqs]: nodes on the way; null: another launch writes the three
  int* path;                             // [seqs, width]: the nodes, then -1
  int* taken;                            // [seqs, width]: what was drawn at each, then -1
  int width;
};

__global__ void __launch_bounds__(CA_THREADS) cache_accept_kernel(const AcceptArgs a) {
  __shared__ int child[CA_MAX_NODES], way[CA_MAX_NODES], n_way;
  __shared__ __align__(16) uint8_t rows[CA_MAX_NODES * CA_COLUMN];
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.y, tid = threadIdx.x;
  const int start = a.seq_q_start[seq], n = min(a.seq_q_len[seq], min(a.width, CA_MAX_NODES)), past = a.seq_kv_len[seq] - a.seq_q_len[seq];
  for (int i = tid; i < n; i += CA_THREADS) child[i] = CA_MAX_NODES;
  __syncthreads();
  for (int i = tid; i < n; i += CA_THREADS) {
    const int p = a.parents[start + i];
    if (p >= 0 && p < i && a.tokens[start + i] == a.drawn[start + p]) atomicMin(&child[p], i);
  }
  __syncthreads();
  if (tid == 0) {
    int k = 0;
    for (int at = 0; at < n; at = child[at]) way[k++] = at;
    n_way = k;
  }
  __syncthreads();
  const int k = n_way;
  if (blockIdx.x == 0 && a.count) {
    for (int i = tid; i < a.width; i += CA_THREADS) {
      a.path[(size_t)seq * a.width + i] = i < k ? way[i] : -1;
      a.taken[(size_t)seq * a.width + i] = i < k ? a.drawn[start + way[i]] : -1;
    }
    if (tid == 0) a.count[seq] = k;
  }
  const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.table_stride;
  const int columns0 = (a.row_bytes[0] + CA_COLUMN - 1) / CA_COLUMN, columns1 = (a.row_bytes[1] + CA_COLUMN - 1) / CA_COLUMN;
  const int columns = columns0 + columns1;
  for (long long job = blockIdx.x; job < (long long)a.pairs * columns; job += gridDim.x) {
    const int pair = (int)(job / columns), c = (int)(job - (long long)pair * columns), which = c >= columns0;
    const int first = (which ? c - columns0 : c) * CA_COLUMN, bytes = min(CA_COLUMN, a.row_bytes[which] - first);
    const int entry = pair / a.kv_heads, kvh = pair - entry * a.kv_heads;
    uint8_t* base = a.store[which] + (size_t)entry * a.entry_rows * a.row_bytes[which] + first;
    auto at = [&](int place) {
      return base + page_row(pages[place / SB_PAGE_TOKENS], kvh, place % SB_PAGE_TOKENS, a.kv_heads, a.row_bytes[which]);
    };
    const int words = bytes / 4;
    for (int idx = tid; idx < k * words; idx += CA_THREADS) {
      const int i = idx / words, w = idx - i * words;
      reinterpret_cast<uint32_t*>(rows)[idx] = reinterpret_cast<const uint32_t*>(at(past + way[i]))[w];
    }
    __syncthreads();
    for (int idx = tid; idx < k * words; idx += CA_THREADS) {
      const int i = idx / words, w = idx - i * words;
      if (way[i] != i) reinterpret_cast<uint32_t*>(at(past + i))[w] = reinterpret_cast<const uint32_t*>(rows)[idx];
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------ pages
//
// Copies items (cache pages, a slot's state) of several tensors [outer, items, item_bytes]: item source[i] to item target[i], for every
// outer index.  The pairs travel in the launch's own arguments, so nothing is uploaded.
#define CP_MAX_TENSORS 16
#define CP_MAX_PAIRS 256
#define CP_THREADS 256

struct CopyArgs {
  uint8_t* base[CP_MAX_TENSORS];
  long long outer[CP_MAX_TENSORS], items[CP_MAX_TENSORS], item_bytes[CP_MAX_TENSORS];
  int source[CP_MAX_PAIRS], target[CP_MAX_PAIRS];
  int tensors, pairs;
};

template <typename V>
__global__ void __launch_bounds__(CP_THREADS) cache_copy_kernel(const __grid_constant__ CopyArgs a) {
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.y, pair = blockIdx.x % a.pairs;
  const long long words = a.item_bytes[t] / (long long)sizeof(V);
  for (long long o = blockIdx.x / a.pairs; o < a.outer[t]; o += gridDim.x / a.pairs) {
    const V* from = reinterpret_cast<const V*>(a.base[t] + (o * a.items[t] + a.source[pair]) * a.item_bytes[t]);
    V* to = reinterpret_cast<V*>(a.base[t] + (o * a.items[t] + a.target[pair]) * a.item_bytes[t]);
    for (long long i = threadIdx.x; i < words; i += CP_THREADS) to[i] = from[i];
  }
}

extern "C" {

int sb_cache_accept_max_nodes() { return CA_MAX_NODES; }

// keys and values [entries, pages, kv_heads, 64, row bytes], row bytes multiples of 4; the step's arrays as in attention_tree.cuh;
// count [seqs], path and taken [seqs, width] or all null.  width: at least every sequence's nodes, at most sb_cache_accept_max_nodes().
int sb_cache_accept(void* keys, void* values, int key_bytes, int value_bytes, int entries, int pages, int kv_heads, const int* block_table,
                    int table_stride, const int* seq_slot, const int* seq_q_start, const int* seq_q_len, const int* seq_kv_len, int seqs,
                    const int* tokens, const int* parents, const int* drawn, int* count, int* path, int* taken, int width,
                    cudaStream_t s) {
  if (seqs == 0) return 0;
  if (key_bytes < 4 || key_bytes % 4 || value_bytes < 4 || value_bytes % 4 || entries < 1 || kv_heads < 1 || pages < 1) return -2;
  if (width < 1 || width > CA_MAX_NODES || seqs > 65535 || (((uintptr_t)keys | (uintptr_t)values) & 3)) return -2;
  if ((long long)entries * kv_heads > 0x7fffffffll) return -2;
  AcceptArgs a;
  a.store[0] = (uint8_t*)keys; a.store[1] = (uint8_t*)values;
  a.row_bytes[0] = key_bytes; a.row_bytes[1] = value_bytes;
  a.entry_rows = (long long)pages * kv_heads * SB_PAGE_TOKENS;
  a.pairs = entries * kv_heads; a.kv_heads = kv_heads;
  a.block_table = block_table; a.table_stride = table_stride;
  a.seq_slot = seq_slot; a.seq_q_start = seq_q_start; a.seq_q_len = seq_q_len; a.seq_kv_len = seq_kv_len;
  a.tokens = tokens; a.parents = parents; a.drawn = drawn;
  a.count = count; a.path = path; a.taken = taken; a.width = width;
  const long long jobs = (long long)a.pairs * ((key_bytes + CA_COLUMN - 1) / CA_COLUMN + (value_bytes + CA_COLUMN - 1) / CA_COLUMN);
  const long long most = 148 * 8 / seqs > 1 ? 148 * 8 / seqs : 1;
  return launch_dependent(cache_accept_kernel, dim3((unsigned)(jobs < most ? jobs : most), seqs), dim3(CA_THREADS), 0, s, a);
}

int sb_cache_copy_max_tensors() { return CP_MAX_TENSORS; }
int sb_cache_copy_max_pairs() { return CP_MAX_PAIRS; }

// tensors: up to 16 of {address, outer, items, item bytes} (host memory, 64-bit each); pairs: up to 256 of {source, target} (host memory,
// 32-bit each, every number below each tensor's items; no target is named twice or is a source).
int sb_cache_copy(const long long* tensors, int n_tensors, const int* pairs, int n_pairs, cudaStream_t s) {
  if (n_tensors == 0 || n_pairs == 0) return 0;
  if (n_tensors < 0 || n_tensors > CP_MAX_TENSORS || n_pairs < 0 || n_pairs > CP_MAX_PAIRS) return -2;
  CopyArgs a = {};
  a.tensors = n_tensors; a.pairs = n_pairs;
  uintptr_t bits = 0;
  long long outer = 1;
  for (int t = 0; t < n_tensors; ++t) {
    a.base[t] = (uint8_t*)(uintptr_t)tensors[4 * t];
    a.outer[t] = tensors[4 * t + 1]; a.items[t] = tensors[4 * t + 2]; a.item_bytes[t] = tensors[4 * t + 3];
    bits |= (uintptr_t)tensors[4 * t] | (uintptr_t)a.item_bytes[t];
    if (a.outer[t] > outer) outer = a.outer[t];
  }
  for (int i = 0; i < n_pairs; ++i) {
    a.source[i] = pairs[2 * i]; a.target[i] = pairs[2 * i + 1];
    for (int t = 0; t < n_tensors; ++t)
      if (a.source[i] < 0 || a.target[i] < 0 || a.source[i] >= a.items[t] || a.target[i] >= a.items[t]) return -2;
  }
  if (outer > 0x7fffffffll / n_pairs) return -2;
  const dim3 grid((unsigned)(n_pairs * outer), n_tensors);
  if (bits % 16 == 0) return launch_dependent(cache_copy_kernel<uint4>, grid, dim3(CP_THREADS), 0, s, a);
  if (bits % 4 == 0) return launch_dependent(cache_copy_kernel<uint32_t>, grid, dim3(CP_THREADS), 0, s, a);
  return launch_dependent(cache_copy_kernel<uint8_t>, grid, dim3(CP_THREADS), 0, s, a);
}

}  // extern "C"
