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
// Every block walks its sequence's tree itself (a few shared-memory steps of a tree's depth; a launch of its own would cost more).  A thread then
// moves one 16-byte column (4 bytes where rows do not allow it) of one entry's keys or values of one key/value head through all rows of the
// way, eight rows on their way at a time: nodes come after their parents, so path[i] >= i grows with i, and what is written at row i has been
// read, or is no row of the way.  What bounds it is the chain of the walk, the page numbers, a read and a write: 4 nodes of one sequence in 36
// layers take 2.7 us, 6 nodes of each of 16 sequences (23.6 MB, worth 3.6 us) 4.6; as blocks that moved 128-byte columns through shared memory one
// after another 49.
#define CA_THREADS 256
#define CA_MAX_NODES 256
#define CA_FLIGHT 8

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

template <typename V>
__global__ void __launch_bounds__(CA_THREADS) cache_accept_kernel(const AcceptArgs a) {
  __shared__ int child[CA_MAX_NODES], way[CA_MAX_NODES], n_way;
  __shared__ long long from[CA_MAX_NODES], to[CA_MAX_NODES];   // rows of the first entry and head
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.y, tid = threadIdx.x;
  const int start = a.seq_q_start[seq], n = min(a.seq_q_len[seq], min(a.width, CA_MAX_NODES)), past = a.seq_kv_len[seq] - a.seq_q_len[seq];
  const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.table_stride;
  // (a thread has one node; its loads do not wait for one another)
  const int parent = tid < n ? a.parents[start + tid] : -1, token = tid < n ? a.tokens[start + tid] : 0;
  child[tid] = CA_MAX_NODES;
  __syncthreads();
  if (parent >= 0 && parent < tid && token == a.drawn[start + parent]) atomicMin(&child[parent], tid);
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
  int first = 0;                                          // the first node that does not stay where it is
  while (first < k && way[first] == first) ++first;
  if (first == k) return;
  if (tid >= first && tid < k) {
    const int src = past + way[tid], dst = past + tid;
    from[tid] = (long long)page_row(pages[src / SB_PAGE_TOKENS], 0, src % SB_PAGE_TOKENS, a.kv_heads, 1);
    to[tid] = (long long)page_row(pages[dst / SB_PAGE_TOKENS], 0, dst % SB_PAGE_TOKENS, a.kv_heads, 1);
  }
  __syncthreads();
  const int columns0 = a.row_bytes[0] / (int)sizeof(V), columns = columns0 + a.row_bytes[1] / (int)sizeof(V);
  for (long long job = (long long)blockIdx.x * CA_THREADS + tid; job < (long long)a.pairs * columns; job += (long long)gridDim.x * CA_THREADS) {
    const int pair = (int)(job / columns), c = (int)(job - (long long)pair * columns), which = c >= columns0;
    const int entry = pair / a.kv_heads, kvh = pair - entry * a.kv_heads, bytes = a.row_bytes[which];
    uint8_t* base = a.store[which] + ((size_t)entry * a.entry_rows + (size_t)kvh * SB_PAGE_TOKENS) * bytes +
                    (size_t)(which ? c - columns0 : c) * sizeof(V);
    for (int i0 = first; i0 < k; i0 += CA_FLIGHT) {
      V v[CA_FLIGHT];
#pragma unroll
      for (int i = 0; i < CA_FLIGHT; ++i)
        if (i0 + i < k) v[i] = *reinterpret_cast<const V*>(base + (size_t)from[i0 + i] * bytes);
#pragma unroll
      for (int i = 0; i < CA_FLIGHT; ++i)
        if (i0 + i < k) *reinterpret_cast<V*>(base + (size_t)to[i0 + i] * bytes) = v[i];
    }
  }
}

// ------------------------------------------------------------------------------------------ pages
//
// Copies items (cache pages, a slot's state) of several tensors [outer, items, item_bytes]: item source[i] to item target[i], for every
// outer index.  The pairs travel in the launch's own arguments, so nothing is uploaded.  A block copies one item, 16 bytes a thread at a time.
// What bounds it is memory: 32 pages of 36 layers (604 MB read and written) take 103 us, 5.9 TB/s.  With few items it is a block's own way: one page of 8 layers of
// 4 heads, 16 blocks of 64 KB in 16 rounds of a load and a store each, takes 4.4 us, where the launch and the walk above take 2.7.
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

// keys and values [entries, pages, kv_heads, 64, row bytes], row bytes multiples of 4; the step's arrays as in attention_tree.cuh;
// count [seqs], path and taken [seqs, width] or all null.  width: at least every sequence's nodes, at most 256.
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
  // 16 bytes a thread where rows allow it; one job a thread until the SMs are full
  const bool wide = (((uintptr_t)keys | (uintptr_t)values | (uintptr_t)key_bytes | (uintptr_t)value_bytes) & 15) == 0;
  const long long jobs = (long long)a.pairs * ((key_bytes + value_bytes) / (wide ? 16 : 4));
  const long long blocks = (jobs + CA_THREADS - 1) / CA_THREADS, most = 148 * 8 / seqs > 1 ? 148 * 8 / seqs : 1;
  const dim3 grid((unsigned)(blocks < most ? blocks : most), seqs);
  return wide ? launch_dependent(cache_accept_kernel<uint4>, grid, dim3(CA_THREADS), 0, s, a)
              : launch_dependent(cache_accept_kernel<uint32_t>, grid, dim3(CA_THREADS), 0, s, a);
}

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
