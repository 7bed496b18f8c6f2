// Attention of the nodes of drafted trees over the paged cache (see attention_tree.cuh): the kernel for every type and size.
//
// A block takes 16 packed rows of one key/value head, four to a warp, and walks its part of the sequence's keys 32 at a time (half a page): keys
// and values are copied to shared memory as they are, a tile ahead; a lane scores one key for the warp's four rows (no sum crosses lanes), the online
// softmax keeps a row's reference in every lane and its sum lane by lane, and for the values the lanes turn to the head's entries.  Everything is
// float; a result is rounded to the working type once.  Up to eight parts of a sequence's keys are the blocks of one cluster and meet in shared
// memory.
//
// What bounds it is the chain of a tile (copy, products, maximum, exponentials, values), about 2 us with one warp a scheduler: 2 sequences of
// 13 nodes of 16 heads behind 300 tokens 33.0 us with copies and products in turn and a second kernel, 17.6 now.
#include "allow_smem.cuh"
#include "attention_tree.cuh"

#define TP_WARPS 4
#define TP_THREADS (TP_WARPS * 32)
#define TP_ROWS 4                       // rows a warp
#define TP_TILE (TP_WARPS * TP_ROWS)
#define TP_KEYS 32
#define TP_CLUSTER_MAX 8

// An aligned piece of BYTES, to shared memory.
template <int BYTES> __device__ __forceinline__ void tp_copy(void* dst, const void* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ float4 tp_open(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 tp_open(const bf16* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ uint32_t tp_peer(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float tp_peer_load(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void tp_cluster_barrier() {
  __syncwarp();                    // (.aligned: a whole warp at once)
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// NI: entries of a head a lane keeps (32 NI >= dim).  wide: dim a multiple of 4 and everything aligned to four entries.
template <typename T, int NI, bool CLUSTER>
__global__ void __launch_bounds__(TP_THREADS) attention_tree_plain_kernel(const TreeArgs a, int wide) {
  extern __shared__ __align__(16) uint8_t tp_smem[];
  const int pitch = ((a.dim + 3) & ~3) + 4;           // rows 16 (8) bytes apart modulo all banks: lanes that read a row each meet none twice
  float* q_sm = reinterpret_cast<float*>(tp_smem);    // [16][pitch]; the results at the end
  T* tiles_sm = reinterpret_cast<T*>(q_sm + TP_TILE * pitch);   // two stages of (keys, values): [32][pitch] each
  __shared__ uint32_t masks[TP_TILE][TREE_MAX_WORDS];
  __shared__ float cl_m[TP_TILE], cl_l[TP_TILE];      // the rows' references and sums (CLUSTER)
  __shared__ int sh_low;
  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.z, seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y - seq * a.kv_heads;
  const int q_len = a.seq_q_len[seq], kv_len = a.seq_kv_len[seq], past = kv_len - q_len, start = a.seq_q_start[seq];
  const int group = a.heads / a.kv_heads;
  const int row0 = blockIdx.x * TP_TILE, n_rows = q_len * group;
  if (row0 >= n_rows) return;                         // (the same in every block of a cluster)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.table_stride;
  const T* q = (const T*)a.q;

  int first[TP_ROWS];                                 // the rows' windows' first places
#pragma unroll
  for (int r = 0; r < TP_ROWS; ++r) {
    const int node = min(row0 + warp * TP_ROWS + r, n_rows - 1) / group;
    first[r] = a.window > 0 ? a.tok_pos[start + node] - a.window + 1 : 0;
  }
  if (a.window > 0) {
    if (threadIdx.x == 0) sh_low = past;
    __syncthreads();
    int low = first[0];
#pragma unroll
    for (int r = 1; r < TP_ROWS; ++r) low = min(low, first[r]);
    if (lane == 0) atomicMin(&sh_low, max(low, 0));
    __syncthreads();
  }
  // tiles of half a page, from the one with the first place any row sees
  const int tile_lo = (a.window > 0 ? sh_low : 0) / TP_KEYS, tiles = (kv_len + TP_KEYS - 1) / TP_KEYS - tile_lo;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int begin = tile_lo + min(split * per, tiles), n_tiles = tile_lo + min((split + 1) * per, tiles) - begin;

  // Whole tiles, whatever lies behind the sequence: it is not seen.
  auto load = [&](int i) {
    const int j0 = (begin + i) * TP_KEYS;
    const size_t from = page_row(pages[j0 / SB_PAGE_TOKENS], kvh, j0 % SB_PAGE_TOKENS, a.kv_heads, a.dim);
    T* to = tiles_sm + (i & 1) * 2 * TP_KEYS * pitch;
    const T* k = (const T*)a.k_store + from;
    const T* v = (const T*)a.v_store + from;
    if (wide) {
      const int pieces = a.dim / 4;
      for (int idx = threadIdx.x; idx < TP_KEYS * pieces; idx += TP_THREADS) {
        const int r = idx / pieces, c = (idx - r * pieces) * 4;
        tp_copy<4 * sizeof(T)>(to + r * pitch + c, k + r * a.dim + c);
        tp_copy<4 * sizeof(T)>(to + (TP_KEYS + r) * pitch + c, v + r * a.dim + c);
      }
    } else {
      for (int idx = threadIdx.x; idx < TP_KEYS * pitch; idx += TP_THREADS) {
        const int r = idx / pitch, c = idx - r * pitch;
        to[idx] = c < a.dim ? k[r * a.dim + c] : from_f<T>(0.f);
        to[TP_KEYS * pitch + idx] = c < a.dim ? v[r * a.dim + c] : from_f<T>(0.f);
      }
    }
  };
  if (n_tiles > 0) load(0);
  asm volatile("cp.async.commit_group;" ::: "memory");

  // the tile's queries (rows behind the last look like the last) and masks
  if (wide) {
    const int pieces = a.dim / 4;
#pragma unroll 4
    for (int idx = threadIdx.x; idx < TP_TILE * pieces; idx += TP_THREADS) {
      const int r = idx / pieces, c = (idx - r * pieces) * 4, row = min(row0 + r, n_rows - 1);
      float4 v = tp_open(q + ((size_t)(start + row / group) * a.heads + kvh * group + row % group) * a.dim + c);
      v.x *= a.scale_log2; v.y *= a.scale_log2; v.z *= a.scale_log2; v.w *= a.scale_log2;
      *reinterpret_cast<float4*>(q_sm + r * pitch + c) = v;
    }
  } else {
    for (int idx = threadIdx.x; idx < TP_TILE * pitch; idx += TP_THREADS) {
      const int r = idx / pitch, d = idx - r * pitch, row = min(row0 + r, n_rows - 1);
      q_sm[idx] = d < a.dim ? to_f<T>(q[((size_t)(start + row / group) * a.heads + kvh * group + row % group) * a.dim + d]) * a.scale_log2 : 0.f;
    }
  }
#pragma unroll
  for (int r = 0; r < TP_ROWS; ++r) {
    const int node = min(row0 + warp * TP_ROWS + r, n_rows - 1) / group;
    if (lane < TREE_MAX_WORDS) masks[warp * TP_ROWS + r][lane] = tree_mask_word(a, start, node, lane, q_len, first[r]);
  }

  float m[TP_ROWS], l[TP_ROWS], acc[TP_ROWS][NI];
#pragma unroll
  for (int r = 0; r < TP_ROWS; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) acc[r][i] = 0.f;
  }
  for (int n = 0; n < n_tiles; ++n) {
    if (n + 1 < n_tiles) load(n + 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const T* k_sm = tiles_sm + (n & 1) * 2 * TP_KEYS * pitch;
    const T* v_sm = k_sm + TP_KEYS * pitch;
    const int j0 = (begin + n) * TP_KEYS;
    float s[TP_ROWS], t[TP_ROWS];
#pragma unroll
    for (int r = 0; r < TP_ROWS; ++r) s[r] = t[r] = 0.f;
    const T* kr = k_sm + lane * pitch;
    const float* qr = q_sm + warp * TP_ROWS * pitch;
#pragma unroll 8
    for (int d = 0; d < a.dim; d += 4) {
      const float4 k = tp_open(kr + d);
#pragma unroll
      for (int r = 0; r < TP_ROWS; ++r) {
        const float4 x = *reinterpret_cast<const float4*>(qr + r * pitch + d);
        s[r] = fmaf(x.x, k.x, s[r]);
        t[r] = fmaf(x.y, k.y, t[r]);
        s[r] = fmaf(x.z, k.z, s[r]);
        t[r] = fmaf(x.w, k.w, t[r]);
      }
    }
    float top[TP_ROWS];
#pragma unroll
    for (int r = 0; r < TP_ROWS; ++r) {
      s[r] += t[r];
      if (j0 + TP_KEYS > past || j0 < first[r]) {     // (what is cached and inside the window is seen)
        const uint32_t view = (uint32_t)tree_view(masks[warp * TP_ROWS + r], first[r], past, kv_len, j0);
        if (!((view >> lane) & 1u)) s[r] = -INFINITY;
      }
      top[r] = s[r];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < TP_ROWS; ++r) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], o));
#pragma unroll
    for (int r = 0; r < TP_ROWS; ++r) {
      const float m_new = fmaxf(m[r], top[r]), base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[r] - base);
      s[r] = exp2f(s[r] - base);
      m[r] = m_new;
      l[r] = l[r] * alpha + s[r];
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[r][i] *= alpha;
    }
#pragma unroll 8
    for (int j = 0; j < TP_KEYS; ++j) {
      float v[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) v[i] = lane + 32 * i < a.dim ? to_f<T>(v_sm[j * pitch + lane + 32 * i]) : 0.f;
#pragma unroll
      for (int r = 0; r < TP_ROWS; ++r) {
        const float p = __shfl_sync(0xffffffffu, s[r], j);
        const bool seen = p != 0.f;                   // (a value that a row does not see may be no number)
#pragma unroll
        for (int i = 0; i < NI; ++i) acc[r][i] = seen ? fmaf(p, v[i], acc[r][i]) : acc[r][i];
      }
    }
    __syncthreads();                                  // the stage may be refilled
  }
#pragma unroll
  for (int r = 0; r < TP_ROWS; ++r) l[r] = warp_sum(l[r]);
  if constexpr (CLUSTER) {
    // the parts of a row lie where its queries were (a warp's own rows); every block joins its share of the rows' entries
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TP_ROWS; ++r) {
      const int at = warp * TP_ROWS + r;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (lane + 32 * i < a.dim) q_sm[at * pitch + lane + 32 * i] = acc[r][i];
      if (lane == 0) {
        cl_m[at] = m[r];
        cl_l[at] = l[r];
      }
    }
    __syncthreads();
    tp_cluster_barrier();
    const int rows_here = min(TP_TILE, n_rows - row0);
    for (int idx = split * TP_THREADS + threadIdx.x; idx < rows_here * a.dim; idx += a.splits * TP_THREADS) {
      const int r = idx / a.dim, d = idx - r * a.dim, row = row0 + r;
      float pm[TP_CLUSTER_MAX], pl[TP_CLUSTER_MAX], px[TP_CLUSTER_MAX];
#pragma unroll
      for (int p = 0; p < TP_CLUSTER_MAX; ++p) {
        if (p < a.splits) {
          pm[p] = tp_peer_load(tp_peer(cl_m + r, p));
          pl[p] = tp_peer_load(tp_peer(cl_l + r, p));
          px[p] = tp_peer_load(tp_peer(q_sm + r * pitch + d, p));
        }
      }
      float high = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
      for (int p = 0; p < TP_CLUSTER_MAX; ++p)
        if (p < a.splits && pl[p] != 0.f) high = fmaxf(high, pm[p]);
#pragma unroll
      for (int p = 0; p < TP_CLUSTER_MAX; ++p) {
        if (p >= a.splits || pl[p] == 0.f) continue;
        const float w = exp2f(pm[p] - high);
        sum = fmaf(pl[p], w, sum);
        o = fmaf(px[p], w, o);
      }
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      ((T*)a.out)[((size_t)(start + row / group) * a.heads + kvh * group + row % group) * a.dim + d] = from_f<T>(o * inv);
    }
    tree_cluster_leave();
  } else
#pragma unroll
  for (int r = 0; r < TP_ROWS; ++r) {
    const int row = row0 + warp * TP_ROWS + r;
    if (row >= n_rows) continue;
    const size_t at = (size_t)(start + row / group) * a.heads + kvh * group + row % group;
    const float inv = l[r] > 0.f ? 1.f / l[r] : l[r] == 0.f ? 0.f : l[r];
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (lane + 32 * i < a.dim) ((T*)a.out)[at * a.dim + lane + 32 * i] = from_f<T>(acc[r][i] * inv);
  }
}

template <typename T, int NI>
static int launch_plain(const TreeArgs& a, int seqs, int max_q_len, cudaStream_t s) {
  const int pitch = ((a.dim + 3) & ~3) + 4, smem = pitch * (TP_TILE * 4 + 4 * TP_KEYS * (int)sizeof(T));
  const bool cluster = a.splits > 1;
  if (smem > 47 * 1024) {
    const int e = cluster ? allow_smem<&attention_tree_plain_kernel<T, NI, true>>(smem) : allow_smem<&attention_tree_plain_kernel<T, NI, false>>(smem);
    if (e) return e;
  }
  const int wide = a.dim % 4 == 0 && (((uintptr_t)a.q | (uintptr_t)a.k_store | (uintptr_t)a.v_store) & (4 * sizeof(T) - 1)) == 0;
  const dim3 grid((max_q_len * (a.heads / a.kv_heads) + TP_TILE - 1) / TP_TILE, a.kv_heads * seqs, a.splits);
  if (cluster)
    return launch_dependent_cluster(attention_tree_plain_kernel<T, NI, true>, grid, dim3(TP_THREADS), smem, s, dim3(1, 1, a.splits), a, wide);
  return launch_dependent(attention_tree_plain_kernel<T, NI, false>, grid, dim3(TP_THREADS), smem, s, a, wide);
}

extern "C" {

// dtype 0 float, 1 bfloat16; dim up to 256; splits 1 to 8.
int sb_attention_tree_plain(int dtype, const void* q, void* out, const void* k_store, const void* v_store, const int* block_table,
                            int table_stride, const int* seq_slot, const int* seq_q_start, const int* seq_q_len, const int* seq_kv_len,
                            const int* tok_pos, const void* mask, int words, int seqs, int max_q_len, int heads, int kv_heads, int dim,
                            float scale, int window, int splits, cudaStream_t s) {
  if (seqs == 0 || max_q_len == 0) return 0;
  if (kv_heads <= 0 || heads % kv_heads || dim < 1 || dim > 256 || words < 1 || splits < 1 || splits > TP_CLUSTER_MAX) return -2;
  if ((long long)seqs * kv_heads > 65535 || max_q_len > 32 * TREE_MAX_WORDS) return -2;
  const TreeArgs a{q, out, k_store, v_store, block_table, table_stride, seq_slot, seq_q_start, seq_q_len, seq_kv_len, tok_pos,
                   (const uint32_t*)mask, words < TREE_MAX_WORDS ? words : TREE_MAX_WORDS, heads, kv_heads, dim, scale * 1.4426950408889634f,
                   window > 0 ? window : 0, splits};
  if (dtype == 0) return dim <= 128 ? launch_plain<float, 4>(a, seqs, max_q_len, s) : launch_plain<float, 8>(a, seqs, max_q_len, s);
  if (dtype == 1) return dim <= 128 ? launch_plain<bf16, 4>(a, seqs, max_q_len, s) : launch_plain<bf16, 8>(a, seqs, max_q_len, s);
  return -1;
}

}  // extern "C"
