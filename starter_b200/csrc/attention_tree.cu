// Attention of the nodes of drafted trees over the paged cache (see attention_tree.cuh): the kernel for every type and size.
//
// A block takes 16 packed rows of one key/value head, four to a warp, and walks its part of the sequence's keys 32 at a time: keys and
// values go to shared memory as floats, a lane scores one key for the warp's four rows (no sum crosses lanes), the online softmax keeps a
// row's reference in every lane and its sum lane by lane, and for the values the lanes turn to the head's entries.  Everything is float;
// a result is rounded to the working type once.
#include "allow_smem.cuh"
#include "attention_tree.cuh"

#define TP_WARPS 4
#define TP_ROWS 4                       // rows a warp
#define TP_TILE (TP_WARPS * TP_ROWS)
#define TP_KEYS 32

template <typename T>
__device__ __forceinline__ void tp_load_rows(float* dst, int pitch, const T* store, const int* pages, int j0, int n, int kvh, int kv_heads,
                                             int dim, bool wide) {
  // n rows of this tile, the others zero: whatever lies in them then adds nothing
  if (wide) {
    const int per = dim / 4;
#pragma unroll 8
    for (int idx = threadIdx.x; idx < TP_KEYS * per; idx += TP_WARPS * 32) {
      const int r = idx / per, c = (idx - r * per) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < n) {
        const T* src = store + page_row(pages[(j0 + r) / SB_PAGE_TOKENS], kvh, (j0 + r) % SB_PAGE_TOKENS, kv_heads, dim) + c;
        if constexpr (sizeof(T) == 4) {
          v = *reinterpret_cast<const float4*>(src);
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(src);
          v = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                          __uint_as_float(w.y & 0xffff0000u));
        }
      }
      *reinterpret_cast<float4*>(dst + r * pitch + c) = v;
    }
  } else {
    for (int idx = threadIdx.x; idx < TP_KEYS * dim; idx += TP_WARPS * 32) {
      const int r = idx / dim, c = idx - r * dim;
      dst[r * pitch + c] =
          r < n ? to_f<T>(store[page_row(pages[(j0 + r) / SB_PAGE_TOKENS], kvh, (j0 + r) % SB_PAGE_TOKENS, kv_heads, dim) + c]) : 0.f;
    }
  }
}

// NI: entries of a head a lane keeps (32 NI >= dim).
template <typename T, int NI>
__global__ void __launch_bounds__(TP_WARPS * 32) attention_tree_plain_kernel(const TreeArgs a, int wide) {
  extern __shared__ __align__(16) float tp_smem[];
  const int pitch = ((a.dim + 3) & ~3) + 4;           // rows 16 bytes apart modulo all banks: lanes that read a row each meet none twice
  float* q_sm = tp_smem;                              // [16][pitch]
  float* k_sm = q_sm + TP_TILE * pitch;               // [32][pitch]
  float* v_sm = k_sm + TP_KEYS * pitch;               // [32][pitch]
  __shared__ uint32_t masks[TP_TILE][TREE_MAX_WORDS];
  __shared__ int sh_low;
  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.z % a.splits, seq = blockIdx.z / a.splits, kvh = blockIdx.y;
  const int q_len = a.seq_q_len[seq], kv_len = a.seq_kv_len[seq], past = kv_len - q_len, start = a.seq_q_start[seq];
  const int group = a.heads / a.kv_heads;
  const int row0 = blockIdx.x * TP_TILE, n_rows = q_len * group;
  if (row0 >= n_rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.table_stride;
  const T* q = (const T*)a.q;

  // the tile's queries (rows behind the last look like the last), zeros in the rows' padding
  if (wide) {
    const int per = a.dim / 4;
#pragma unroll 4
    for (int idx = threadIdx.x; idx < TP_TILE * per; idx += TP_WARPS * 32) {
      const int r = idx / per, c = (idx - r * per) * 4, row = min(row0 + r, n_rows - 1);
      const T* src = q + ((size_t)(start + row / group) * a.heads + kvh * group + row % group) * a.dim + c;
      float4 v;
      if constexpr (sizeof(T) == 4) {
        v = *reinterpret_cast<const float4*>(src);
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(src);
        v = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
      }
      v.x *= a.scale_log2; v.y *= a.scale_log2; v.z *= a.scale_log2; v.w *= a.scale_log2;
      *reinterpret_cast<float4*>(q_sm + r * pitch + c) = v;
    }
  } else {
    for (int idx = threadIdx.x; idx < (TP_TILE + 2 * TP_KEYS) * pitch; idx += TP_WARPS * 32) tp_smem[idx] = 0.f;
    __syncthreads();
    for (int idx = threadIdx.x; idx < TP_TILE * a.dim; idx += TP_WARPS * 32) {
      const int r = idx / a.dim, d = idx - r * a.dim, row = min(row0 + r, n_rows - 1);
      q_sm[r * pitch + d] = to_f<T>(q[((size_t)(start + row / group) * a.heads + kvh * group + row % group) * a.dim + d]) * a.scale_log2;
    }
  }
  // the rows' masks and windows
  int first[TP_ROWS];
#pragma unroll
  for (int r = 0; r < TP_ROWS; ++r) {
    const int node = min(row0 + warp * TP_ROWS + r, n_rows - 1) / group;
    first[r] = a.window > 0 ? a.tok_pos[start + node] - a.window + 1 : 0;
    if (lane < TREE_MAX_WORDS) masks[warp * TP_ROWS + r][lane] = tree_mask_word(a, start, node, lane, q_len, first[r]);
  }
  if (threadIdx.x == 0) sh_low = a.window > 0 ? past : 0;
  __syncthreads();
  if (a.window > 0) {
    int low = first[0];
#pragma unroll
    for (int r = 1; r < TP_ROWS; ++r) low = min(low, first[r]);
    if (lane == 0) atomicMin(&sh_low, max(low, 0));
    __syncthreads();
  }
  const int lowest = sh_low;                          // the first place any of the tile's rows sees
  const int tiles = (kv_len - lowest + TP_KEYS - 1) / TP_KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int begin = lowest + split * per * TP_KEYS, end = min(begin + per * TP_KEYS, kv_len);

  float m[TP_ROWS], l[TP_ROWS], acc[TP_ROWS][NI];
#pragma unroll
  for (int r = 0; r < TP_ROWS; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) acc[r][i] = 0.f;
  }
  for (int j0 = begin; j0 < end; j0 += TP_KEYS) {
    __syncthreads();                                  // the tile before has been read
    const int n = min(TP_KEYS, end - j0);
    tp_load_rows<T>(k_sm, pitch, (const T*)a.k_store, pages, j0, n, kvh, a.kv_heads, a.dim, wide);
    tp_load_rows<T>(v_sm, pitch, (const T*)a.v_store, pages, j0, n, kvh, a.kv_heads, a.dim, wide);
    __syncthreads();
    float s[TP_ROWS];
#pragma unroll
    for (int r = 0; r < TP_ROWS; ++r) s[r] = 0.f;
    const float* kr = k_sm + lane * pitch;
    const float* qr = q_sm + warp * TP_ROWS * pitch;
    for (int d = 0; d < a.dim; d += 4) {
      const float4 k = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
      for (int r = 0; r < TP_ROWS; ++r) {
        const float4 x = *reinterpret_cast<const float4*>(qr + r * pitch + d);
        s[r] = fmaf(x.x, k.x, s[r]);
        s[r] = fmaf(x.y, k.y, s[r]);
        s[r] = fmaf(x.z, k.z, s[r]);
        s[r] = fmaf(x.w, k.w, s[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < TP_ROWS; ++r) {
      if (lane >= n) s[r] = -INFINITY;
      if (j0 + n > past || j0 < first[r]) {           // (what is cached and inside the window is seen)
        const uint32_t view = (uint32_t)tree_view(masks[warp * TP_ROWS + r], first[r], past, kv_len, j0);
        if (!((view >> lane) & 1u)) s[r] = -INFINITY;
      }
      const float m_new = fmaxf(m[r], warp_max(s[r]));
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[r] - base);
      s[r] = exp2f(s[r] - base);
      m[r] = m_new;
      l[r] = l[r] * alpha + s[r];
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[r][i] *= alpha;
    }
    for (int j = 0; j < n; ++j) {
      float v[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) v[i] = lane + 32 * i < a.dim ? v_sm[j * pitch + lane + 32 * i] : 0.f;
#pragma unroll
      for (int r = 0; r < TP_ROWS; ++r) {
        const float p = __shfl_sync(0xffffffffu, s[r], j);
        if (p != 0.f) {                               // (a value that a row does not see may be no number)
#pragma unroll
          for (int i = 0; i < NI; ++i) acc[r][i] = fmaf(p, v[i], acc[r][i]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < TP_ROWS; ++r) {
    const int row = row0 + warp * TP_ROWS + r;
    const float sum = warp_sum(l[r]);
    if (row >= n_rows) continue;
    const size_t at = (size_t)(start + row / group) * a.heads + kvh * group + row % group;
    if (a.splits == 1) {
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (lane + 32 * i < a.dim) ((T*)a.out)[at * a.dim + lane + 32 * i] = from_f<T>(acc[r][i] * inv);
    } else {
      const size_t p = at * a.splits + split;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (lane + 32 * i < a.dim) a.part_acc[p * a.dim + lane + 32 * i] = acc[r][i];
      if (lane == 0) {
        a.part_ml[2 * p] = m[r];
        a.part_ml[2 * p + 1] = sum;
      }
    }
  }
}

template <typename T, int NI>
static int launch_plain(const TreeArgs& a, int seqs, int max_q_len, cudaStream_t s) {
  const int pitch = ((a.dim + 3) & ~3) + 4, smem = (TP_TILE + 2 * TP_KEYS) * pitch * 4;
  if (smem > 48 * 1024) {
    const int e = allow_smem<&attention_tree_plain_kernel<T, NI>>(smem);
    if (e) return e;
  }
  const int bytes = sizeof(T) == 4 ? 16 : 8;
  const int wide = a.dim % 4 == 0 && (((uintptr_t)a.q | (uintptr_t)a.k_store | (uintptr_t)a.v_store) & (bytes - 1)) == 0;
  const dim3 grid((max_q_len * (a.heads / a.kv_heads) + TP_TILE - 1) / TP_TILE, a.kv_heads, seqs * a.splits);
  int rc = launch_dependent(attention_tree_plain_kernel<T, NI>, grid, dim3(TP_WARPS * 32), smem, s, a, wide);
  if (rc || a.splits == 1) return rc;
  return launch_dependent(attention_tree_join_kernel<T>, dim3(max_q_len, seqs, (a.heads + 3) / 4), dim3(128), 0, s, a);
}

extern "C" {

// dtype 0 float, 1 bfloat16; dim up to 256; splits 1 to 32, with part_acc and part_ml (see TreeArgs) from 2 on.
int sb_attention_tree_plain(int dtype, const void* q, void* out, const void* k_store, const void* v_store, const int* block_table,
                            int table_stride, const int* seq_slot, const int* seq_q_start, const int* seq_q_len, const int* seq_kv_len,
                            const int* tok_pos, const void* mask, int words, int seqs, int max_q_len, int heads, int kv_heads, int dim,
                            float scale, int window, int splits, float* part_acc, float* part_ml, cudaStream_t s) {
  if (seqs == 0 || max_q_len == 0) return 0;
  if (kv_heads <= 0 || heads % kv_heads || dim < 1 || dim > 256 || words < 1 || splits < 1 || splits > 32) return -2;
  if ((long long)seqs * splits > 65535 || kv_heads > 65535 || seqs > 65535) return -2;
  if (splits > 1 && (!part_acc || !part_ml)) return -2;
  const TreeArgs a{q, out, k_store, v_store, block_table, table_stride, seq_slot, seq_q_start, seq_q_len, seq_kv_len, tok_pos,
                   (const uint32_t*)mask, words, heads, kv_heads, dim, scale * 1.4426950408889634f, window > 0 ? window : 0, splits,
                   part_acc, part_ml};
  if (dtype == 0) return dim <= 128 ? launch_plain<float, 4>(a, seqs, max_q_len, s) : launch_plain<float, 8>(a, seqs, max_q_len, s);
  if (dtype == 1) return dim <= 128 ? launch_plain<bf16, 4>(a, seqs, max_q_len, s) : launch_plain<bf16, 8>(a, seqs, max_q_len, s);
  return -1;
}

}  // extern "C"
