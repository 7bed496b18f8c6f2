// Attention of the nodes of drafted trees over the paged cache (see attention_tree.cuh) on mma.sync, in bfloat16: steps whose rows are few.
//
// A block takes a tile of 16 or 32 packed rows of one key/value head and walks its part of the sequence's pages.  WR warps own
// 16 rows each; the 4 / WR warps that own the same rows take a share of a page's 64 keys each.  A page (keys and values) goes to a ring of
// three shared-memory stages by 16-byte asynchronous copies, two pages ahead, swizzled for ldmatrix; S = Q K^T, the online softmax in
// float, P rounded to bfloat16 (half a step of 8 bits of each weight, what the prompt kernels do), O += P V.  The warps' results meet in
// shared memory; up to eight parts of a sequence's keys are the blocks of one cluster and meet there.
//
// Places behind the sequence or in front of what a window leaves are copied as zeros, so whatever lies there adds nothing.  A value
// that is no number must reach the rows that see it and no others, though a weight of zero times it is none: on pages that some row
// does not see whole such entries are taken out of the tile, and put onto the results of the rows that see them at the end.
//
// What bounds it, with few rows, is the chain of dependent steps: 5 nodes of one sequence behind 1,500 tokens (32 heads of 128 on 8: 128 blocks of
// three pages) take 8.3 us, where their 6 MB are worth 1: 1.3 us to the first copy (the step's arrays, the table), 1.3 until the page is there, 0.5 a page, 0.9
// for the meeting of the warps, 1.8 for that of the blocks.  A second kernel for the meeting of more parts cost more than it gave (16,000 tokens, 16
// rows: 29.6 us as 8 parts, 26.9 as 32 and a second kernel, but 2 more at 1,500); tiles of 64 rows were slower than two of 32 wherever tried.
// With many rows it is mma.sync's issue: 128 pairs of 64 rows behind 1,500 tokens 38 us.
#include "allow_smem.cuh"
#include "attention_tree.cuh"

#define TM_WARPS 4
#define TM_THREADS (TM_WARPS * 32)
#define TM_STAGES 3
#define TM_CLUSTER_MAX 8
#define TM_MAX_NODES 256

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes, or zeros where `bytes` is 0.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t peer_u32(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float peer_load(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 peer_load2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();                    // (.aligned: a whole warp at once)
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Byte offset of 16-byte piece `chunk` of row `row` of a [rows][D] bfloat16 tile whose rows' pieces are swizzled.
template <int D> __device__ __forceinline__ int tile_offset(int row, int chunk) {
  constexpr int C = D / 8;
  const int sw = C >= 8 ? (row & 7) : ((row / (8 / C)) % C);
  return row * D * 2 + ((chunk ^ sw) << 4);
}
__device__ __forceinline__ bool no_number(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }

template <int D, int WR, bool CLUSTER>
__global__ void __launch_bounds__(TM_THREADS, D > 64 ? 2 : 4) attention_tree_mma_kernel(const TreeArgs a) {
  constexpr int C = D / 8, PAGE_BYTES = SB_PAGE_TOKENS * D * 2, STAGE_BYTES = 2 * PAGE_BYTES;
  constexpr int KSTEPS = D / 16, NBLK = D / 8;
  constexpr int WK = TM_WARPS / WR, KEYS = SB_PAGE_TOKENS / WK, KBLK = KEYS / 8, ROWS = 16 * WR;
  constexpr int DP = D + 8;                             // floats between rows of the warps' results
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* q_tile = smem;                               // [ROWS][D]
  uint8_t* ring = smem + ROWS * D * 2;                  // stages of (keys, values); the results at the end
  __shared__ uint32_t sh_mask[ROWS][TREE_MAX_WORDS];    // of the tile's nodes (at most one a row)
  __shared__ int sh_first[ROWS];                        // their windows' first places
  __shared__ float sh_m[WK][ROWS], sh_l[WK][ROWS];
  __shared__ float2 cl_ml[ROWS];                        // the block's reference and sum of a row
  __shared__ int sh_bad;

  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.z, seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y - seq * a.kv_heads;
  const int q_len = a.seq_q_len[seq], kv_len = a.seq_kv_len[seq], past = kv_len - q_len, start = a.seq_q_start[seq];
  const int group = a.heads / a.kv_heads, row0 = blockIdx.x * ROWS, n_rows = q_len * group;
  if (row0 >= n_rows) return;                           // (the same in every block of a cluster)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wr = warp % WR, wk = warp / WR;
  const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.table_stride;
  const int node0 = row0 / group, n_nodes = (min(row0 + ROWS, n_rows) - 1) / group - node0 + 1;

  if (tid == 0) sh_bad = 0;
  const int low = tree_low(a, past), high = tree_high(a, past, kv_len);
  const int first_page = low / SB_PAGE_TOKENS, end_page = (kv_len + SB_PAGE_TOKENS - 1) / SB_PAGE_TOKENS;
  const int per_split = (end_page - first_page + a.splits - 1) / a.splits;
  const int p_begin = first_page + split * per_split, n_pages = max(min(p_begin + per_split, end_page) - p_begin, 0);

  auto load_page = [&](int i) {
    if (i < n_pages) {
      const int j0 = (p_begin + i) * SB_PAGE_TOKENS;
      const size_t base = page_row(pages[p_begin + i], kvh, 0, a.kv_heads, D);
      uint8_t* dst = ring + (size_t)(i % TM_STAGES) * STAGE_BYTES;
      for (int idx = tid; idx < SB_PAGE_TOKENS * C; idx += TM_THREADS) {
        const int r = idx / C, c = idx % C, bytes = j0 + r >= low && j0 + r < kv_len ? 16 : 0;
        cp_async16(dst + tile_offset<D>(r, c), (const bf16*)a.k_store + base + (size_t)idx * 8, bytes);
        cp_async16(dst + PAGE_BYTES + tile_offset<D>(r, c), (const bf16*)a.v_store + base + (size_t)idx * 8, bytes);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < TM_STAGES - 1; ++i) load_page(i);

  // ---- while those are on their way: the tile's nodes' masks and queries (rows behind the last are zero)
  constexpr int WORDS = ROWS * TREE_MAX_WORDS / TM_THREADS;
  uint32_t words[WORDS];
  int firsts[WORDS];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    const int n = min((tid + i * TM_THREADS) / TREE_MAX_WORDS, n_nodes - 1);
    firsts[i] = a.window > 0 ? a.tok_pos[start + node0 + n] - a.window + 1 : 0;
    words[i] = tree_mask_word(a, start, node0 + n, tid % TREE_MAX_WORDS, q_len, firsts[i], past);
  }
#pragma unroll
  for (int idx0 = 0; idx0 < ROWS * C; idx0 += TM_THREADS) {
    const int idx = idx0 + tid, r = idx / C, c = idx % C, row = row0 + r;
    if (idx >= ROWS * C) break;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < n_rows)
      v = *reinterpret_cast<const uint4*>((const bf16*)a.q + ((size_t)(start + row / group) * a.heads + kvh * group + row % group) * D + c * 8);
    *reinterpret_cast<uint4*>(q_tile + tile_offset<D>(r, c)) = v;
  }
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    const int n = (tid + i * TM_THREADS) / TREE_MAX_WORDS;
    sh_mask[n][tid % TREE_MAX_WORDS] = words[i];
    if (tid % TREE_MAX_WORDS == 0) sh_first[n] = firsts[i];
  }
  __syncthreads();

  uint32_t qf[KSTEPS][4];
  {
    const int r = wr * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk)
      ldmatrix_x4(smem_u32(q_tile + tile_offset<D>(r, 2 * kk + (lane >> 4))), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
  }
  // the thread's two rows' nodes in the tile (rows behind the last look like the last)
  int node[2], from[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    node[h] = min(row0 + wr * 16 + (lane >> 2) + 8 * h, n_rows - 1) / group - node0;
    from[h] = sh_first[node[h]];
  }
  float o[NBLK][4];
#pragma unroll
  for (int n = 0; n < NBLK; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

  for (int i = 0; i < n_pages; ++i) {
    load_page(i + TM_STAGES - 1);
    cp_wait<TM_STAGES - 1>();
    __syncthreads();
    const uint8_t* kt = ring + (size_t)(i % TM_STAGES) * STAGE_BYTES;
    uint8_t* vt = const_cast<uint8_t*>(kt) + PAGE_BYTES;
    const int page_j0 = (p_begin + i) * SB_PAGE_TOKENS;
    // some row does not see all of the page
    const bool edge = page_j0 + SB_PAGE_TOKENS > past || page_j0 < high;
    if (edge) {
      int bad = 0;
      for (int idx = tid; idx < SB_PAGE_TOKENS * C; idx += TM_THREADS) {
        uint4* at = reinterpret_cast<uint4*>(vt + idx * 16);
        uint32_t w[4] = {at->x, at->y, at->z, at->w};
        int here = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (no_number(w[e])) { w[e] &= 0xffff0000u; here = 1; }
          if (no_number(w[e] >> 16)) { w[e] &= 0xffffu; here = 1; }
        }
        if (here) { *at = make_uint4(w[0], w[1], w[2], w[3]); bad = 1; }
      }
      if (bad) sh_bad = 1;
      __syncthreads();
    }

    float s[KBLK][4];
#pragma unroll
    for (int nb = 0; nb < KBLK; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
#pragma unroll
      for (int nb = 0; nb < KBLK; nb += 2) {
        uint32_t b0, b1, b2, b3;
        const int key = wk * KEYS + nb * 8 + (lane & 7) + (lane >> 4) * 8;
        ldmatrix_x4(smem_u32(kt + tile_offset<D>(key, 2 * kk + ((lane >> 3) & 1))), b0, b1, b2, b3);
        mma_bf16(s[nb], qf[kk], b0, b1);
        mma_bf16(s[nb + 1], qf[kk], b2, b3);
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nb = 0; nb < KBLK; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nb][e] *= a.scale_log2;
    if (edge) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // (shifted so that the thread's own columns of a block of eight keys come first)
        const uint64_t view = tree_view(sh_mask[node[h]], from[h], past, kv_len, page_j0) >> (wk * KEYS + (lane & 3) * 2);
        const uint32_t lo = (uint32_t)view, hi = (uint32_t)(view >> 32);
#pragma unroll
        for (int nb = 0; nb < KBLK; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!(((nb < 4 ? lo : hi) >> (nb % 4 * 8 + e)) & 1u)) s[nb][2 * h + e] = -INFINITY;
      }
    }
#pragma unroll
    for (int nb = 0; nb < KBLK; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[nb][e]);
    float alpha[2], base[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      const float m_new = fmaxf(m_run[h], mx[h]);
      base[h] = m_new == -INFINITY ? 0.f : m_new;
      alpha[h] = fast_exp2(m_run[h] - base[h]);
      m_run[h] = m_new;
      l_run[h] *= alpha[h];
    }
#pragma unroll
    for (int n = 0; n < NBLK; ++n) { o[n][0] *= alpha[0]; o[n][1] *= alpha[0]; o[n][2] *= alpha[1]; o[n][3] *= alpha[1]; }
#pragma unroll
    for (int kb = 0; kb < KEYS / 16; ++kb) {
      uint32_t pf[4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float* x = s[2 * kb + t];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = fast_exp2(x[e] - base[e >> 1]);
          l_run[e >> 1] += x[e];
        }
        pf[2 * t] = pack_bf16(x[0], x[1]);
        pf[2 * t + 1] = pack_bf16(x[2], x[3]);
      }
#pragma unroll
      for (int n = 0; n < NBLK; n += 2) {
        uint32_t b0, b1, b2, b3;
        const int key = wk * KEYS + kb * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
        ldmatrix_x4_trans(smem_u32(vt + tile_offset<D>(key, n + (lane >> 4))), b0, b1, b2, b3);
        mma_bf16(o[n], pf, b0, b1);
        mma_bf16(o[n + 1], pf, b2, b3);
      }
    }
    __syncthreads();                                    // the stage may be refilled
  }
  cp_wait<0>();
  __syncthreads();

  // ---- the warps' parts of a row meet in the ring's place: [WK][ROWS][DP]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
  }
  float* sh_o = reinterpret_cast<float*>(ring);
  {
    const int r = wr * 16 + (lane >> 2);
    if ((lane & 3) == 0) {
      sh_m[wk][r] = m_run[0]; sh_m[wk][r + 8] = m_run[1];
      sh_l[wk][r] = l_run[0]; sh_l[wk][r + 8] = l_run[1];
    }
    float* to = sh_o + ((size_t)wk * ROWS + r) * DP + (lane & 3) * 2;
#pragma unroll
    for (int n = 0; n < NBLK; ++n) {
      *reinterpret_cast<float2*>(to + n * 8) = make_float2(o[n][0], o[n][1]);
      *reinterpret_cast<float2*>(to + 8 * DP + n * 8) = make_float2(o[n][2], o[n][3]);
    }
  }
  __syncthreads();
  const int rows_here = min(ROWS, n_rows - row0);
  auto out_at = [&](int r) {
    const int row = row0 + r;
    return ((size_t)(start + row / group) * a.heads + kvh * group + row % group);
  };
  if (tid < rows_here) {                                // the weights the warps' parts of a row have in it (negative: a part without keys)
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) top = fmaxf(top, sh_l[w][tid] != 0.f ? sh_m[w][tid] : -INFINITY);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float l = sh_l[w][tid], f = l == 0.f ? -1.f : WK == 1 ? 1.f : fast_exp2(sh_m[w][tid] - top);
      if (l != 0.f) sum = fmaf(l, f, sum);
      sh_m[w][tid] = f;
    }
    cl_ml[tid] = make_float2(top, sum);
  }
  __syncthreads();
  // (every entry of a row is one thread's from here to the end of the block; loads in front of stores, which they could be for all the compiler knows)
  constexpr int FLIGHT = 4;
  for (int idx0 = tid; idx0 < rows_here * (D / 2); idx0 += FLIGHT * TM_THREADS) {
    float2 x[FLIGHT];
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) {
      const int idx = idx0 + u * TM_THREADS, r = min(idx / (D / 2), ROWS - 1), d = idx % (D / 2) * 2;
      x[u] = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float f = sh_m[w][r];
        const float2 y = *reinterpret_cast<const float2*>(sh_o + ((size_t)w * ROWS + r) * DP + d);
        // (a weight below zero is not, one that is no number is)
        x[u].x = f < 0.f ? x[u].x : fmaf(y.x, f, x[u].x);
        x[u].y = f < 0.f ? x[u].y : fmaf(y.y, f, x[u].y);
      }
    }
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) {
      const int idx = idx0 + u * TM_THREADS, r = idx / (D / 2), d = idx % (D / 2) * 2;
      if (r < rows_here) *reinterpret_cast<float2*>(sh_o + (size_t)r * DP + d) = x[u];
    }
  }
  if (sh_bad) {                                         // what was taken out of the tiles, to the rows that see it
#pragma unroll 1
    for (int idx = tid; idx < rows_here * (D / 2); idx += TM_THREADS) {
      const int r = idx / (D / 2), d = (idx - r * (D / 2)) * 2, n = (row0 + r) / group - node0;
      float2* x = reinterpret_cast<float2*>(sh_o + (size_t)r * DP + d);
      for (int j = p_begin * SB_PAGE_TOKENS; j < min((p_begin + n_pages) * SB_PAGE_TOKENS, kv_len); ++j) {
        if (!(tree_view(sh_mask[n], sh_first[n], past, kv_len, j) & 1ull)) continue;
        const uint32_t v = *reinterpret_cast<const uint32_t*>((const bf16*)a.v_store + page_row(pages[j / SB_PAGE_TOKENS], kvh, j % SB_PAGE_TOKENS, a.kv_heads, D) + d);
        if (no_number(v)) x->x += __uint_as_float(v << 16);
        if (no_number(v >> 16)) x->y += __uint_as_float(v & 0xffff0000u);
      }
    }
  }
  if constexpr (!CLUSTER) {
    for (int idx = tid; idx < rows_here * (D / 2); idx += TM_THREADS) {
      const int r = idx / (D / 2), d = (idx - r * (D / 2)) * 2;
      const float sum = cl_ml[r].y, inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      const float2 x = *reinterpret_cast<const float2*>(sh_o + (size_t)r * DP + d);
      *reinterpret_cast<uint32_t*>((bf16*)a.out + out_at(r) * D + d) = pack_bf16(x.x * inv, x.y * inv);
    }
  }
  if constexpr (CLUSTER) {
    // every block joins its share of the tile's rows, reading the others' parts
    cluster_barrier();
    for (int idx = split * TM_THREADS + tid; idx < rows_here * (D / 2); idx += a.splits * TM_THREADS) {
      const int r = idx / (D / 2), d = (idx - r * (D / 2)) * 2;
      float2 ml[TM_CLUSTER_MAX], x[TM_CLUSTER_MAX];
#pragma unroll
      for (int p = 0; p < TM_CLUSTER_MAX; ++p) {
        if (p < a.splits) {
          ml[p] = peer_load2(peer_u32(cl_ml + r, p));
          x[p] = peer_load2(peer_u32(sh_o + (size_t)r * DP + d, p));
        }
      }
      float top = -INFINITY, sum = 0.f;
      float2 y = make_float2(0.f, 0.f);
#pragma unroll
      for (int p = 0; p < TM_CLUSTER_MAX; ++p)
        if (p < a.splits && ml[p].y != 0.f) top = fmaxf(top, ml[p].x);
#pragma unroll
      for (int p = 0; p < TM_CLUSTER_MAX; ++p) {
        if (p >= a.splits || ml[p].y == 0.f) continue;
        const float f = fast_exp2(ml[p].x - top);
        sum = fmaf(ml[p].y, f, sum);
        y.x = fmaf(x[p].x, f, y.x);
        y.y = fmaf(x[p].y, f, y.y);
      }
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      *reinterpret_cast<uint32_t*>((bf16*)a.out + out_at(r) * D + d) = pack_bf16(y.x * inv, y.y * inv);
    }
    tree_cluster_leave();
  }
}

template <int D, int WR>
static int launch_rows(const TreeArgs& a, int seqs, int max_q_len, cudaStream_t s) {
  constexpr int RING = TM_STAGES * 2 * SB_PAGE_TOKENS * D * 2, JOIN = 64 * (D + 8) * 4;
  const int smem = 16 * WR * D * 2 + (RING > JOIN ? RING : JOIN);
  const bool cluster = a.splits > 1;
  const int e = cluster ? allow_smem<&attention_tree_mma_kernel<D, WR, true>>(smem) : allow_smem<&attention_tree_mma_kernel<D, WR, false>>(smem);
  if (e) return e;
  const dim3 grid((max_q_len * (a.heads / a.kv_heads) + 16 * WR - 1) / (16 * WR), a.kv_heads * seqs, a.splits);
  if (cluster)
    return launch_dependent_cluster(attention_tree_mma_kernel<D, WR, true>, grid, dim3(TM_THREADS), smem, s, dim3(1, 1, a.splits), a);
  return launch_dependent(attention_tree_mma_kernel<D, WR, false>, grid, dim3(TM_THREADS), smem, s, a);
}

template <int D>
static int launch(const TreeArgs& a, int seqs, int max_q_len, int row_warps, cudaStream_t s) {
  return row_warps == 1 ? launch_rows<D, 1>(a, seqs, max_q_len, s) : launch_rows<D, 2>(a, seqs, max_q_len, s);
}

extern "C" {

// bfloat16, dim 16, 32, 64 or 128 (-2 otherwise), q and the stores 16-byte aligned; row_warps 1 or 2: tiles of 16 or 32 rows.  splits 1 to 8.
int sb_attention_tree_mma(const void* q, void* out, const void* k_store, const void* v_store, const int* block_table, int table_stride,
                          const int* seq_slot, const int* seq_q_start, const int* seq_q_len, const int* seq_kv_len, const int* tok_pos,
                          const void* mask, int words, int seqs, int max_q_len, int heads, int kv_heads, int dim, float scale, int window,
                          int splits, int row_warps, cudaStream_t s) {
  if (seqs == 0 || max_q_len == 0) return 0;
  if (kv_heads <= 0 || heads % kv_heads || words < 1 || splits < 1 || splits > TM_CLUSTER_MAX) return -2;
  if (row_warps != 1 && row_warps != 2) return -2;
  if ((long long)seqs * kv_heads > 65535 || max_q_len > TM_MAX_NODES) return -2;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_store | (uintptr_t)v_store) & 15) return -2;
  const TreeArgs a{q, out, k_store, v_store, block_table, table_stride, seq_slot, seq_q_start, seq_q_len, seq_kv_len, tok_pos,
                   (const uint32_t*)mask, words, words < TREE_MAX_WORDS ? words : TREE_MAX_WORDS, heads, kv_heads, dim,
                   scale * 1.4426950408889634f, window > 0 ? window : 0, splits};
  switch (dim) {
    case 16: return launch<16>(a, seqs, max_q_len, row_warps, s);
    case 32: return launch<32>(a, seqs, max_q_len, row_warps, s);
    case 64: return launch<64>(a, seqs, max_q_len, row_warps, s);
    case 128: return launch<128>(a, seqs, max_q_len, row_warps, s);
    default: return -2;
  }
}

}  // extern "C"
