// Log probabilities of given tokens and entropies straight from hidden rows and the head, in bfloat16: x = h w^T is formed tile by tile on the
// tensor cores and goes no further than tensor memory.
//
// The product is the persistent CTA-pair kernel of gemm_prompt_tcgen05.cu (tiles of 256 rows x `bn` of the vocabulary, a ring of TMA stages,
// two accumulators in tensor memory).  Its epilogue reads a tile's row of logits, 32 at a time, into the running statistics of
// logprob_stats.cuh, caps them first where asked, and leaves (m, L, T) of the row and tile in scratch memory; the thread that meets
// the row's own token leaves its logit.  A second kernel joins a row's tiles.  The logits of 2,048 rows over 151,936 tokens would be 1.2 GB
// written and read again; the scratch is 16 bytes a row and tile.
//
// What bounds it is the product: those 2,048 rows of 2,560 entries (1.59 TFLOP) take 1.10 ms, 1.45 PFLOP/s, and the epilogue hides behind it.  333 rows over
// 32,768 tokens (width 2,048) take 49 us where 27 would do: they fill two row tiles of 256, and the tiles come in rounds of 74 pairs.  With the
// vocabulary on the tile's rows and these rows on its columns the padding goes, but a row's statistics then cross lanes: about a tenth less, not kept.
//
// Every wait on an mbarrier gives up after a time limit, raises bit 4 of *status and lets both CTAs drain, free their tensor memory and return.
#include "allow_smem.cuh"
#include "cta_pair.cuh"
#include "logprob_stats.cuh"
#include "tensor_map.cuh"

struct ScoreArgs {
  int rows, vocab, k_dim;
  int bn;                   // vocabulary entries a tile
  int stages, m_tiles, n_tiles, group_m;
  const int* tokens;        // [rows]
  float cap;                // 0: none
  float4* part;             // [n_tiles][rows]: m, L, T of a row's logits in a tile
  float* logit;             // [rows]: that of the row's token
  int* status;
  unsigned long long wait_limit_ns;
  int withhold_kblock;      // >= 0 (tests only): the first CTA leaves out its weight copy of this k-block of its first tile
};

// Which tile is the t-th: row tiles in groups of `group_m`, inside a group the row tiles of one vocabulary tile next to each other, so that
// a weight tile is read from memory once a group and from L2 by the group's other row tiles.
__device__ __forceinline__ void sc_tile(const ScoreArgs& a, int t, int& mt, int& nt) {
  const int per_group = a.group_m * a.n_tiles, g = t / per_group, r = t - g * per_group, here = min(a.group_m, a.m_tiles - g * a.group_m);
  nt = r / here;
  mt = g * a.group_m + (r - nt * here);
}

template <bool CAP>
__global__ void __launch_bounds__(PG_THREADS, 1)
score_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w, const ScoreArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full_bar[PG_MAX_STAGES], empty_bar[PG_MAX_STAGES], acc_full[2], acc_empty[2], drain_bar;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;

  const int STAGES = a.stages, half_n = a.bn / 2, STAGE_BYTES = PG_A_BYTES + half_n * PG_TILE_K * 2;
  const uint64_t limit = a.wait_limit_ns;
  // the warp's number as a value the compiler knows to be the same in every lane
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = pg_cluster_rank();               // 0: the CTA that issues the MMAs
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, tiles = a.m_tiles * a.n_tiles;
  const int n_kb = (a.k_dim + PG_TILE_K - 1) / PG_TILE_K;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 8); }
    mbar_init(&drain_bar, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) pg_tmem_alloc(&tmem_holder, PG_TMEM_COLS);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  pg_cluster_sync();     // both CTAs' barriers exist before either signals the other's
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  pdl_trigger();
  const uint32_t tmem = tmem_holder;
  volatile int* abort = &abort_flag;

  if (warp == 0) {
    // ---------------- producer: the warp walks the ring together, one elected lane issues the copies
    const bool elected = elect_one();
    pdl_wait();
    int it = 0, s = 0;
    uint32_t parity = 1;          // flips at every wrap of the ring; the first pass waits for nothing
    bool gave_up = false;
    for (int t = pair; t < tiles && !gave_up; t += n_pairs) {
      int mt, nt;
      sc_tile(a, t, mt, nt);
      const int m0 = mt * PG_TILE_M + (int)rank * PG_ROWS_PER_CTA, w0 = nt * a.bn + (int)rank * half_n;
      const bool withheld_tile = rank == 0 && t == pair;
      for (int kb = 0; kb < n_kb; ++kb, ++it) {
        if (it >= STAGES && !__all_sync(0xffffffffu, mbar_wait(&empty_bar[s], parity, abort, limit))) { gave_up = true; break; }
        uint8_t* stage = smem + (size_t)s * STAGE_BYTES;
        const uint32_t full = pg_in_cta(smem_u32(&full_bar[s]), 0);
        if (elected) {
          if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * STAGE_BYTES);
          pg_tma_load(stage, &map_h, full, kb * PG_TILE_K, m0);
          if (!(withheld_tile && kb == a.withhold_kblock)) pg_tma_load(stage + PG_A_BYTES, &map_w, full, kb * PG_TILE_K, w0);
        }
        if (++s == STAGES) { s = 0; parity ^= 1; }
      }
    }
    if (*abort && elected) {
      // copies still in flight write into this CTA's shared memory: give them time to land
      const uint64_t begun = now_ns();
      while (now_ns() - begun < 100000ull) {}
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer: the warp of the first CTA, one elected lane issues
    if (rank == 0) {
      const bool elected = elect_one();
      const uint32_t idesc = pg_instr_desc(a.bn);
      int i = 0, s = 0;
      uint32_t parity = 0;
      bool gave_up = false;
      for (int t = pair; t < tiles && !gave_up; t += n_pairs, ++i) {
        const int b = i & 1;
        if (i >= 2 && !__all_sync(0xffffffffu, mbar_wait(&acc_empty[b], ((i >> 1) - 1) & 1, abort, limit))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + (uint32_t)b * PG_ACC_STRIDE;
        for (int kb = 0; kb < n_kb; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[s], parity, abort, limit))) { gave_up = true; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t a_addr = smem_u32(smem + (size_t)s * STAGE_BYTES);
          const uint64_t a_desc = smem_desc(a_addr), b_desc = smem_desc(a_addr + PG_A_BYTES);
          if (elected) {
#pragma unroll
            for (int k = 0; k < PG_TILE_K / 16; ++k) pg_mma(d, a_desc + 2 * k, b_desc + 2 * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
            pg_commit_both(&empty_bar[s]);
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; parity ^= 1; }
        }
        if (!gave_up && elected) pg_commit_both(&acc_full[b]);
        __syncwarp();
      }
      if (*abort && elected) {
        // the MMAs issued so far must be over before tensor memory and shared memory are given up
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&drain_bar)) : "memory");
        const uint64_t begun = now_ns();
        while (!mbar_try(&drain_bar, 0) && now_ns() - begun < limit) {}
      }
    }
  } else {
    // ---------------- epilogue: warps 2..5 own the tensor-memory lane quarters 2, 3, 0, 1; thread = row
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t empty0 = pg_in_cta(smem_u32(&acc_empty[0]), 0), empty1 = pg_in_cta(smem_u32(&acc_empty[1]), 0);
    pdl_wait();   // before the first store: the scratch may be memory an earlier kernel still reads
    int i = 0;
    for (int t = pair; t < tiles; t += n_pairs, ++i) {
      const int b = i & 1;
      int mt, nt;
      sc_tile(a, t, mt, nt);
      const int grow = mt * PG_TILE_M + (int)rank * PG_ROWS_PER_CTA + row, col0 = nt * a.bn;
      const bool valid = grow < a.rows;
      const int token = valid ? a.tokens[grow] - col0 : -1;     // its place in this tile
      // the whole warp goes on or the whole warp stops: the reads below are warp-wide instructions
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (i >> 1) & 1, abort, limit))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = lane_base + (uint32_t)b * PG_ACC_STRIDE;
      const int n_chunks = a.bn / 32;
      Stats st{-INFINITY, 0.f, 0.f};
#pragma unroll 1
      for (int c = 0; c < n_chunks; ++c) {
        float v[32];
        pg_tmem_load32(acc + c * 32, v);
        if (c == n_chunks - 1) {
          // this warp has read all it needs of the accumulator: the tensor cores may have it back
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) pg_arrive_cluster(b ? empty1 : empty0);
        }
        if (CAP) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = a.cap * tanhf(v[j] / a.cap);
        }
        if (__any_sync(0xffffffffu, (unsigned)(token - 32 * c) < 32u)) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (token == 32 * c + j) a.logit[grow] = v[j];
        }
        const int left = a.vocab - col0 - 32 * c;         // entries from here on (behind them the weights read as zeros)
        if (left < 32) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j >= left) v[j] = -INFINITY;
        }
        float mx = v[0];
#pragma unroll
        for (int j = 1; j < 32; ++j) mx = fmaxf(mx, v[j]);
        if (mx > st.m) st = lp_join(st, Stats{mx, 0.f, 0.f});
        const float base = st.m == -INFINITY ? 0.f : st.m;
        float l0 = 0.f, l1 = 0.f, t0 = 0.f, t1 = 0.f;
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float d0 = v[j] - base, d1 = v[j + 1] - base, p0 = lp_exp(d0), p1 = lp_exp(d1);
          l0 += p0;
          l1 += p1;
          t0 = fmaf(p0, fmaxf(d0, -1e30f), t0);
          t1 = fmaf(p1, fmaxf(d1, -1e30f), t1);
        }
        st.l += l0 + l1;
        st.t += t0 + t1;
      }
      if (valid) a.part[(size_t)nt * a.rows + grow] = make_float4(st.m, st.l, st.t, 0.f);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  pg_cluster_sync();     // nobody leaves while the other CTA may still signal its barriers or read its memory
  if (warp == 1) pg_tmem_free(tmem, PG_TMEM_COLS);
  if (threadIdx.x == 0 && abort_flag && a.status) atomicOr(a.status, 4);
}

// Joins a row's tiles: a block takes eight rows, 32 threads each (a warp reads 128 bytes of four tiles at once).
#define SJ_ROWS 8
__global__ void __launch_bounds__(256) score_join_kernel(const float4* part, const float* logit, const int* tokens, int rows, int vocab, int n_tiles,
                                                         float* given, float* entropy, int* status) {
  __shared__ Stats sh[32][SJ_ROWS];
  pdl_trigger();
  pdl_wait();
  SB_BEHIND_WAIT(part);
  SB_BEHIND_WAIT(logit);
  SB_BEHIND_WAIT(tokens);
  const int r = threadIdx.x % SJ_ROWS, g = threadIdx.x / SJ_ROWS, row = blockIdx.x * SJ_ROWS + r;
  Stats st{-INFINITY, 0.f, 0.f};
  if (row < rows) {
#pragma unroll 4
    for (int nt = g; nt < n_tiles; nt += 32) {
      const float4 p = part[(size_t)nt * rows + row];
      st = lp_join(st, Stats{p.x, p.y, p.z});
    }
  }
  sh[g][r] = st;
  __syncthreads();
  for (int half = 16; half > 0; half >>= 1) {
    if (g < half) sh[g][r] = lp_join(sh[g][r], sh[g + half][r]);
    __syncthreads();
  }
  if (g == 0 && row < rows) {
    st = sh[0][r];
    const float log_l = st.l > 0.f ? logf(st.l) : NAN;    // (a sum that is no number makes a row whose probabilities are none)
    const int t = tokens[row];
    float x = 0.f;
    if (t >= vocab) {
      x = NAN;
      if (status) atomicOr(status, 1);
    } else if (t >= 0) {
      x = (logit[row] - st.m) - log_l;
    }
    given[row] = x;
    entropy[row] = log_l - st.t / st.l;
  }
}

// ------------------------------------------------------------------------------------------ host

static int sc_pairs() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms / 2;
}

// Vocabulary entries a tile: the least time on the busiest CTA pair, rounds of tiles times what a tile of that width takes (a k-block costs
// about 150 ns and 1.04 ns a weight row).
static int sc_bn(int rows, int vocab, int pairs) {
  const int m_tiles = (rows + PG_TILE_M - 1) / PG_TILE_M;
  int bn = 0;
  long long best = -1;
  for (int cand = 256; cand >= 128; cand -= 32) {
    const long long tiles = (long long)m_tiles * ((vocab + cand - 1) / cand);
    const long long cost = ((tiles + pairs - 1) / pairs) * (cand + 144);
    if (best < 0 || cost < best) { best = cost; bn = cand; }
  }
  return bn;
}

template <bool CAP>
static int sc_launch(const CUtensorMap& mh, const CUtensorMap& mw, const ScoreArgs& a, int pairs, int smem, cudaStream_t s) {
  const int e = allow_smem<&score_kernel<CAP>>(smem);
  if (e) return e;
  return launch_dependent_cluster(score_kernel<CAP>, dim3(2 * pairs), dim3(PG_THREADS), smem, s, dim3(2, 1, 1), mh, mw, a);
}

static unsigned long long next_limit_ns = TC_WAIT_LIMIT_NS;
static int next_withhold = -1;

extern "C" {

// For tests of the give-up path: the NEXT sb_score launch leaves out one weight copy (k-block `kblock` of the first tile of every first
// CTA) and its waits give up after `limit_ns`; it must return with bit 4 of *status set.
void sb_score_withhold(int kblock, unsigned long long limit_ns) {
  next_withhold = kblock;
  next_limit_ns = limit_ns ? limit_ns : TC_WAIT_LIMIT_NS;
}

// How many floats of scratch sb_score needs: 16 bytes a row and vocabulary tile, and a logit a row.
long long sb_score_scratch(int rows, int vocab) {
  const int bn = sc_bn(rows, vocab, sc_pairs());
  return 4ll * ((vocab + bn - 1) / bn) * rows + rows;
}

// h [rows, k_dim] and w [vocab, k_dim] bfloat16, row-major, 16-byte aligned, k_dim a multiple of 8; tokens [rows] (negative: none; vocab or
// more: bit 1 of *status); cap 0: none; given, entropy [rows]; scratch: 16-byte aligned, sb_score_scratch(rows, vocab) floats.
int sb_score(const void* h, const void* w, const int* tokens, int rows, int vocab, int k_dim, float cap, float* given, float* entropy,
             float* scratch, int* status, cudaStream_t s) {
  if (rows == 0) return 0;
  if (vocab < 1 || k_dim < 8 || k_dim % 8 || cap < 0.f) return -2;
  if (((uintptr_t)h | (uintptr_t)w | (uintptr_t)scratch) & 15) return -2;
  int pairs = sc_pairs();
  if (pairs < 1) return -2;
  ScoreArgs a;
  a.bn = sc_bn(rows, vocab, pairs);
  a.rows = rows; a.vocab = vocab; a.k_dim = k_dim;
  a.m_tiles = (rows + PG_TILE_M - 1) / PG_TILE_M; a.n_tiles = (vocab + a.bn - 1) / a.bn;
  const int stage_bytes = PG_A_BYTES + a.bn / 2 * PG_TILE_K * 2;
  a.stages = (227 * 1024 - 1024 - 1024) / stage_bytes;
  if (a.stages > PG_MAX_STAGES) a.stages = PG_MAX_STAGES;
  if ((long long)a.m_tiles * a.n_tiles > 0x7fffffffll) return -2;
  if (a.m_tiles * a.n_tiles < pairs) pairs = a.m_tiles * a.n_tiles;
  // a group's rows of h (group_m x 256 x k x 2 bytes) should stay in L2 beside the weights passing by
  long long group_m = (48ll << 20) / (512ll * k_dim);
  group_m = group_m > 16 ? 16 : group_m < 1 ? 1 : group_m;
  a.group_m = group_m > a.m_tiles ? a.m_tiles : (int)group_m;
  a.tokens = tokens; a.cap = cap; a.status = status;
  a.part = (float4*)scratch; a.logit = scratch + 4ll * a.n_tiles * rows;
  a.wait_limit_ns = next_limit_ns; a.withhold_kblock = next_withhold;
  next_limit_ns = TC_WAIT_LIMIT_NS;
  next_withhold = -1;
  CUtensorMap mh, mw;
  int rc = sb_make_map(&mh, h, rows, k_dim, PG_ROWS_PER_CTA);
  if (rc) return rc;
  rc = sb_make_map(&mw, w, vocab, k_dim, a.bn / 2);
  if (rc) return rc;
  const int smem = a.stages * stage_bytes + 1024;
  rc = cap > 0.f ? sc_launch<true>(mh, mw, a, pairs, smem, s) : sc_launch<false>(mh, mw, a, pairs, smem, s);
  if (rc) return rc;
  return launch_dependent(score_join_kernel, dim3((rows + SJ_ROWS - 1) / SJ_ROWS), dim3(256), 0, s, (const float4*)a.part, (const float*)a.logit, tokens,
                          rows, vocab, a.n_tiles, given, entropy, status);
}

}  // extern "C"
