// Attention of the nodes of drafted trees over the paged cache (see attention_tree.cuh): the kernel for every type and size.
//
// A block takes 16 packed rows of one key/value head and walks its part of the sequence's keys 32 at a time (half a page): keys and values are
// copied to shared memory as they are, a tile ahead.  A warp takes 8 of a tile's keys for all rows: a lane scores one key for four rows (five loads
// of 16 bytes for 16 products, none of which meets another's bank), the online softmax of a row crosses eight lanes, and for the values a
// lane turns to four entries of the head, for all rows (a load of 16 bytes and four broadcast ones for 64 products).  The warps keep
// references, sums and outputs of their own, which meet at the end.  Everything is float; a result is rounded to the working type
// once.  Up to eight parts of a sequence's keys are the blocks of one cluster and meet in shared memory.
//
// What bounds it: 2 sequences of 13 nodes of 16 heads behind 300 tokens, 256 blocks of two tiles, take 15.6 us: 5 until the first tile is there (the
// step's arrays, the page's number, the page, which the four blocks of a head's rows all read), 2.9 a tile (the products of queries and
// keys 1.2, of weights and values 1.1, most of it the shared memory's rate), 3.5 for the meeting of the blocks.  Keys a lane each and
// rows a warp each read the tile four times over: 17.2; copies and products in turn and a second kernel for the meeting: 33.0.
#include "allow_smem.cuh"
#include "attention_tree.cuh"

#define TP_WARPS 4
#define TP_THREADS (TP_WARPS * 32)
#define TP_TILE 16                      // rows
#define TP_KEYS 32
#define TP_WARP_KEYS (TP_KEYS / TP_WARPS)
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
__device__ __forceinline__ float4 tp_peer_load4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void tp_cluster_barrier() {
  __syncwarp();                    // (.aligned: a whole warp at once)
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Four entries of a result: at once, or the first `n` of them one by one.
__device__ __forceinline__ void tp_close(float* p, const float4& v, bool at_once, int n) {
  if (at_once) { *reinterpret_cast<float4*>(p) = v; return; }
  p[0] = v.x;
  if (n > 1) p[1] = v.y;
  if (n > 2) p[2] = v.z;
  if (n > 3) p[3] = v.w;
}
__device__ __forceinline__ void tp_close(bf16* p, const float4& v, bool at_once, int n) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
  if (at_once) { *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi)); return; }
  p[0] = lo.x;
  if (n > 1) p[1] = lo.y;
  if (n > 2) p[2] = hi.x;
  if (n > 3) p[3] = hi.y;
}

// NJ: pieces of four entries of a head a lane keeps (128 NJ >= dim).  wide: dim a multiple of 4 and everything aligned to four entries.
template <typename T, int NJ, bool CLUSTER>
__global__ void __launch_bounds__(TP_THREADS, NJ == 1 ? 3 : 1) attention_tree_plain_kernel(const TreeArgs a, int wide) {
  extern __shared__ __align__(16) uint8_t tp_smem[];
  const int padded = (a.dim + 3) & ~3, pitch = padded + 4;   // rows 16 (8) bytes apart modulo all banks: lanes that read a row each meet none twice
  float* q_sm = reinterpret_cast<float*>(tp_smem);    // [16][pitch]
  T* tiles_sm = reinterpret_cast<T*>(q_sm + TP_TILE * pitch);   // two stages of (keys, values): [32][pitch] each; the warps' results at the end
  __shared__ __align__(16) float p_sm[TP_WARPS][TP_WARP_KEYS][TP_TILE + 4], alpha_sm[TP_WARPS][TP_TILE];
  __shared__ uint32_t masks[TP_TILE][TREE_MAX_WORDS];
  __shared__ int firsts[TP_TILE];                     // the rows' windows' first places
  __shared__ float sh_m[TP_WARPS][TP_TILE], sh_l[TP_WARPS][TP_TILE];
  __shared__ float cl_m[TP_TILE], cl_l[TP_TILE];      // the rows' references and sums
  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.z, seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y - seq * a.kv_heads;
  const int q_len = a.seq_q_len[seq], kv_len = a.seq_kv_len[seq], past = kv_len - q_len, start = a.seq_q_start[seq];
  const int group = a.heads / a.kv_heads;
  const int row0 = blockIdx.x * TP_TILE, n_rows = q_len * group;
  if (row0 >= n_rows) return;                         // (the same in every block of a cluster)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.table_stride;
  const T* q = (const T*)a.q;

  // tiles of half a page, from the one with the first place any row sees
  const int tile_lo = tree_low(a, past) / TP_KEYS, tiles = (kv_len + TP_KEYS - 1) / TP_KEYS - tile_lo;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int begin = tile_lo + min(split * per, tiles), n_tiles = tile_lo + min((split + 1) * per, tiles) - begin;

  // Whole tiles, whatever lies behind the sequence: it is not seen.  A warp copies every fourth row.
  auto load = [&](int i) {
    const int j0 = (begin + i) * TP_KEYS;
    const size_t from = page_row(pages[j0 / SB_PAGE_TOKENS], kvh, j0 % SB_PAGE_TOKENS, a.kv_heads, a.dim);
    T* to = tiles_sm + (i & 1) * 2 * TP_KEYS * pitch;
    const T* k = (const T*)a.k_store + from;
    const T* v = (const T*)a.v_store + from;
    for (int r = warp; r < TP_KEYS; r += TP_WARPS) {
      if (wide) {
        for (int c = 4 * lane; c < a.dim; c += 128) {
          tp_copy<4 * sizeof(T)>(to + r * pitch + c, k + r * a.dim + c);
          tp_copy<4 * sizeof(T)>(to + (TP_KEYS + r) * pitch + c, v + r * a.dim + c);
        }
      } else {
        for (int c = lane; c < padded; c += 32) {
          to[r * pitch + c] = c < a.dim ? k[r * a.dim + c] : from_f<T>(0.f);
          to[(TP_KEYS + r) * pitch + c] = c < a.dim ? v[r * a.dim + c] : from_f<T>(0.f);
        }
      }
    }
  };
  if (n_tiles > 0) load(0);
  asm volatile("cp.async.commit_group;" ::: "memory");

  // the rows' masks, a word a thread, and queries (rows behind the last look like the last)
  static_assert(TP_TILE * TREE_MAX_WORDS == TP_THREADS, "a word of the masks for every thread");
  const int my_node = min(row0 + tid / TREE_MAX_WORDS, n_rows - 1) / group, my_first = a.window > 0 ? a.tok_pos[start + my_node] - a.window + 1 : 0;
  const uint32_t word = tree_mask_word(a, start, my_node, tid % TREE_MAX_WORDS, q_len, my_first, past);
#pragma unroll
  for (int n = 0; n < TP_TILE / TP_WARPS; ++n) {
    const int r = warp + n * TP_WARPS, row = min(row0 + r, n_rows - 1);
    const T* from = q + ((size_t)(start + row / group) * a.heads + kvh * group + row % group) * a.dim;
    if (wide) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int c = 4 * lane + 128 * j;
        if (c >= a.dim) break;
        float4 v = tp_open(from + c);
        v.x *= a.scale_log2; v.y *= a.scale_log2; v.z *= a.scale_log2; v.w *= a.scale_log2;
        *reinterpret_cast<float4*>(q_sm + r * pitch + c) = v;
      }
    } else {
      for (int c = lane; c < padded; c += 32) q_sm[r * pitch + c] = c < a.dim ? to_f<T>(from[c]) * a.scale_log2 : 0.f;
    }
  }
  masks[tid / TREE_MAX_WORDS][tid % TREE_MAX_WORDS] = word;
  if (tid % TREE_MAX_WORDS == 0) firsts[tid / TREE_MAX_WORDS] = my_first;

  // A lane's key of a tile and its rows: group, group + 4, ...
  const int key = warp * TP_WARP_KEYS + (lane & 7), row_of = lane >> 3;
  float m[4], l[4], acc[TP_TILE][4 * NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
#pragma unroll
  for (int r = 0; r < TP_TILE; ++r)
#pragma unroll
    for (int e = 0; e < 4 * NJ; ++e) acc[r][e] = 0.f;
  for (int n = 0; n < n_tiles; ++n) {
    if (n + 1 < n_tiles) load(n + 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const T* k_sm = tiles_sm + (n & 1) * 2 * TP_KEYS * pitch;
    const T* v_sm = k_sm + TP_KEYS * pitch;
    const int j0 = (begin + n) * TP_KEYS;
    float s[4], t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = t[i] = 0.f;
    const T* kr = k_sm + key * pitch;
    const float* qr = q_sm + row_of * pitch;
#pragma unroll 8
    for (int d = 0; d < padded; d += 4) {
      const float4 k = tp_open(kr + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(qr + 4 * i * pitch + d);
        s[i] = fmaf(x.x, k.x, s[i]);
        t[i] = fmaf(x.y, k.y, t[i]);
        s[i] = fmaf(x.z, k.z, s[i]);
        t[i] = fmaf(x.w, k.w, t[i]);
      }
    }
    bool moved = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row_of + 4 * i, first = firsts[r];
      bool hidden = false;
      s[i] += t[i];
      if (j0 + TP_KEYS > past || j0 < first) {        // (what is cached and inside the window is seen)
        const uint32_t view = (uint32_t)tree_view(masks[r], first, past, kv_len, j0);
        hidden = !((view >> key) & 1u);
        if (hidden) s[i] = -INFINITY;
      }
      float top = s[i];
#pragma unroll
      for (int o = 1; o < TP_WARP_KEYS; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float m_new = fmaxf(m[i], top), base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[i] - base);
      s[i] = hidden ? -0.f : exp2f(s[i] - base);      // (a key that is not seen is told from one whose weight is too small for a float)
      moved |= m_new > m[i];
      m[i] = m_new;
      l[i] = l[i] * alpha + s[i];
      p_sm[warp][lane & 7][r] = s[i];
      if ((lane & 7) == 0) alpha_sm[warp][r] = alpha;
    }
    __syncwarp();
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int r = 0; r < TP_TILE; r += 4) {
        const float4 f = *reinterpret_cast<const float4*>(&alpha_sm[warp][r]);
#pragma unroll
        for (int e = 0; e < 4 * NJ; ++e) { acc[r][e] *= f.x; acc[r + 1][e] *= f.y; acc[r + 2][e] *= f.z; acc[r + 3][e] *= f.w; }
      }
    }
#pragma unroll 2
    for (int j = 0; j < TP_WARP_KEYS; ++j) {
      float v[4 * NJ];
      bool numbers = true;
#pragma unroll
      for (int e = 0; e < NJ; ++e) {
        const int d = 4 * lane + 128 * e;
        const float4 x = d < padded ? tp_open(v_sm + (warp * TP_WARP_KEYS + j) * pitch + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[4 * e] = x.x; v[4 * e + 1] = x.y; v[4 * e + 2] = x.z; v[4 * e + 3] = x.w;
        numbers &= fabsf(x.x) < INFINITY && fabsf(x.y) < INFINITY && fabsf(x.z) < INFINITY && fabsf(x.w) < INFINITY;
      }
      float p[TP_TILE];
#pragma unroll
      for (int r = 0; r < TP_TILE; r += 4) *reinterpret_cast<float4*>(p + r) = *reinterpret_cast<const float4*>(&p_sm[warp][j][r]);
      if (__all_sync(0xffffffffu, numbers)) {
#pragma unroll
        for (int r = 0; r < TP_TILE; ++r)
#pragma unroll
          for (int e = 0; e < 4 * NJ; ++e) acc[r][e] = fmaf(p[r], v[e], acc[r][e]);
      } else {                                        // (one that is no number reaches the rows that see it, however small their weights, and no others)
#pragma unroll
        for (int r = 0; r < TP_TILE; ++r)
#pragma unroll
          for (int e = 0; e < 4 * NJ; ++e) acc[r][e] = __float_as_uint(p[r]) != 0x80000000u ? fmaf(p[r], v[e], acc[r][e]) : acc[r][e];
      }
    }
    __syncthreads();                                  // the stage may be refilled
  }

  // ---- the warps' parts meet where the tiles were: [warps][16][pitch]
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 1; o < TP_WARP_KEYS; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    if ((lane & 7) == 0) {
      sh_m[warp][row_of + 4 * i] = m[i];
      sh_l[warp][row_of + 4 * i] = l[i];
    }
  }
  float* o_sm = reinterpret_cast<float*>(tiles_sm);
#pragma unroll
  for (int r = 0; r < TP_TILE; ++r)
#pragma unroll
    for (int e = 0; e < NJ; ++e)
      if (4 * lane + 128 * e < padded)
        *reinterpret_cast<float4*>(o_sm + (warp * TP_TILE + r) * pitch + 4 * lane + 128 * e) =
            make_float4(acc[r][4 * e], acc[r][4 * e + 1], acc[r][4 * e + 2], acc[r][4 * e + 3]);
  __syncthreads();
  if (tid < TP_TILE) {                                // the weights the warps' parts of a row have in it (negative: a part without keys)
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < TP_WARPS; ++w) top = fmaxf(top, sh_l[w][tid] != 0.f ? sh_m[w][tid] : -INFINITY);
#pragma unroll
    for (int w = 0; w < TP_WARPS; ++w) {
      const float part = sh_l[w][tid], f = part == 0.f ? -1.f : exp2f(sh_m[w][tid] - top);
      if (part != 0.f) sum = fmaf(part, f, sum);
      sh_m[w][tid] = f;
    }
    cl_m[tid] = top;
    cl_l[tid] = sum;
  }
  __syncthreads();
  const int rows_here = min(TP_TILE, n_rows - row0), pieces = padded / 4;
  auto out_at = [&](int r, int d) {
    const int row = row0 + r;
    return (T*)a.out + ((size_t)(start + row / group) * a.heads + kvh * group + row % group) * a.dim + d;
  };
  for (int idx = tid; idx < rows_here * pieces; idx += TP_THREADS) {
    const int r = idx / pieces, d = (idx - r * pieces) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < TP_WARPS; ++w) {
      const float f = sh_m[w][r];
      const float4 y = *reinterpret_cast<const float4*>(o_sm + (w * TP_TILE + r) * pitch + d);
      if (!(f < 0.f)) { x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y); x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w); }
    }
    if constexpr (CLUSTER) {
      *reinterpret_cast<float4*>(q_sm + r * pitch + d) = x;
    } else {
      const float sum = cl_l[r], inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
      tp_close(out_at(r, d), x, wide, a.dim - d);
    }
  }
  if constexpr (CLUSTER) {
    // the blocks' parts of a row lie where its queries were; every block joins its share of them
    tp_cluster_barrier();
    for (int idx = split * TP_THREADS + tid; idx < rows_here * pieces; idx += a.splits * TP_THREADS) {
      const int r = idx / pieces, d = (idx - r * pieces) * 4;
      float pm[TP_CLUSTER_MAX], pl[TP_CLUSTER_MAX];
      float4 px[TP_CLUSTER_MAX];
#pragma unroll
      for (int p = 0; p < TP_CLUSTER_MAX; ++p) {
        if (p < a.splits) {
          pm[p] = tp_peer_load(tp_peer(cl_m + r, p));
          pl[p] = tp_peer_load(tp_peer(cl_l + r, p));
          px[p] = tp_peer_load4(tp_peer(q_sm + r * pitch + d, p));
        }
      }
      float high = -INFINITY, sum = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < TP_CLUSTER_MAX; ++p)
        if (p < a.splits && pl[p] != 0.f) high = fmaxf(high, pm[p]);
#pragma unroll
      for (int p = 0; p < TP_CLUSTER_MAX; ++p) {
        if (p >= a.splits || pl[p] == 0.f) continue;
        const float w = exp2f(pm[p] - high);
        sum = fmaf(pl[p], w, sum);
        o.x = fmaf(px[p].x, w, o.x); o.y = fmaf(px[p].y, w, o.y); o.z = fmaf(px[p].z, w, o.z); o.w = fmaf(px[p].w, w, o.w);
      }
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
      tp_close(out_at(r, d), o, wide, a.dim - d);
    }
    tree_cluster_leave();
  }
}

template <typename T, int NJ>
static int launch_plain(const TreeArgs& a, int seqs, int max_q_len, cudaStream_t s) {
  const int pitch = ((a.dim + 3) & ~3) + 4, smem = pitch * (TP_TILE * 4 + 4 * TP_KEYS * (int)sizeof(T));
  static_assert(TP_WARPS * TP_TILE * 4 <= 4 * TP_KEYS * (int)sizeof(T), "the warps' results fit where the tiles were");
  const bool cluster = a.splits > 1;
  if (smem > 40 * 1024) {
    const int e = cluster ? allow_smem<&attention_tree_plain_kernel<T, NJ, true>>(smem) : allow_smem<&attention_tree_plain_kernel<T, NJ, false>>(smem);
    if (e) return e;
  }
  const int wide = a.dim % 4 == 0 && (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k_store | (uintptr_t)a.v_store) & (4 * sizeof(T) - 1)) == 0;
  const dim3 grid((max_q_len * (a.heads / a.kv_heads) + TP_TILE - 1) / TP_TILE, a.kv_heads * seqs, a.splits);
  if (cluster)
    return launch_dependent_cluster(attention_tree_plain_kernel<T, NJ, true>, grid, dim3(TP_THREADS), smem, s, dim3(1, 1, a.splits), a, wide);
  return launch_dependent(attention_tree_plain_kernel<T, NJ, false>, grid, dim3(TP_THREADS), smem, s, a, wide);
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
                   (const uint32_t*)mask, words, words < TREE_MAX_WORDS ? words : TREE_MAX_WORDS, heads, kv_heads, dim, scale * 1.4426950408889634f,
                   window > 0 ? window : 0, splits};
  if (dtype == 0) return dim <= 128 ? launch_plain<float, 1>(a, seqs, max_q_len, s) : launch_plain<float, 2>(a, seqs, max_q_len, s);
  if (dtype == 1) return dim <= 128 ? launch_plain<bf16, 1>(a, seqs, max_q_len, s) : launch_plain<bf16, 2>(a, seqs, max_q_len, s);
  return -1;
}

}  // extern "C"
