// Attention of the nodes of drafted trees over the paged cache (see attention_tree.cuh) on the fifth-generation tensor cores, in bfloat16:
// steps whose trees have many rows.
//
// A block takes 256 packed rows of one key/value head as two tiles of 128 and walks the sequence's keys in steps of 128 (two pages):
//     S  = Q K^T     M = 128 rows, N = 128 keys,  K = head_dim        (Q and K K-major)
//     O += P V       M = 128 rows, N = head_dim,  K = 128 keys        (V as it lies in the cache, "MN-major")
// with S and O of both tiles in tensor memory.  Warps 0-3 and 4-7 are the softmax of tile 0 and 1 (thread = row = tensor-memory lane), warp 8
// brings keys and values by TMA, warps 9 and 10 issue the products of tile 0 and 1: the schedule of the prompt attention
// (attention_prefill_tc.cu), with all rows of a sequence's tree on one copy of its keys.  The queries of a tile lie in up to 128 pieces of
// the packed rows; a softmax warp puts its own rows into shared memory.
//
// A row's view of a page is 64 bits: ones for what is cached (from its window's first place on), then the bits of its mask, shifted to where
// the nodes begin in the page.  Only pages that some row does not see whole are masked.  On those a value that is no number is taken out of
// the tile before its product (it must not reach rows that do not see it, though their weight is zero) and put onto the results of the rows
// that see it at the end.
//
// Few blocks over many keys: `splits` CTAs, a cluster, walk a part of a block's keys each and meet through distributed shared memory.
//
// What bounds it is the softmax: a step of 128 keys takes 1.07 us with one tile and 1.5 with two, of which the exponentials of 2 x 128 x 128
// scores are worth 1.07 at 16 a clock and the products 0.55.  16 sequences of 64 nodes behind up to 4,096 tokens each (32 heads of 128 on
// 8, 128 blocks) take 65 us, 207 MB and 41 GFLOP that are worth 31: the longest sequence's 33 steps, 50 us, behind which the other SMs rest.  Tried
// and slower: a cubic in place of every fourth exponential (1.54 us a step) or every second (1.80); sixteen softmax warps, two threads a row (1.78: the
// weights no longer fit in registers in front of the wait for the product before); both tiles on the same 128 rows where there are no more, every
// second step each (16 x 32 nodes 57.7 us against 49.7: a copy's way from memory lies in every step).
//
// Every wait on an mbarrier gives up after WAIT_LIMIT_NS, raises bit 16 of *status and lets the block drain its copies, free its tensor memory
// and return.
#include <cuda.h>

#include "allow_smem.cuh"
#include "attention_tc.cuh"
#include "attention_tree.cuh"
#include "tensor_map.cuh"

#define TT_BK 128
#define TT_THREADS 352
#define TT_ROWS (2 * TC_BQ)
#define TT_MAX_NODES 256
#define TT_MAX_SPLITS 8
// tree_view of a mask in registers: every word is taken by its number.
__device__ __forceinline__ uint64_t tt_view(const uint32_t* bits, int first, int past, int q_len, int j0) {
  uint64_t view = 0;
#pragma unroll
  for (int w = 0; w < TREE_MAX_WORDS; ++w) {
    const int at = past + 32 * w - j0;                    // where its first node stands in the page
    if (at > -32 && at < 64) view |= at >= 0 ? (uint64_t)bits[w] << at : (uint64_t)(bits[w] >> -at);
  }
  const int cached = past - j0, end = cached + q_len, hidden = min(first, past) - j0;
  if (cached > 0) view |= cached < 64 ? (1ull << cached) - 1 : ~0ull;
  if (end < 64) view &= end > 0 ? (1ull << end) - 1 : 0ull;          // places behind the sequence
  if (hidden > 0) view &= hidden < 64 ? ~0ull << hidden : 0ull;      // cached places in front of the window
  return view;
}
// 8 consecutive 32-bit columns of this thread's TMEM lane, there and back (few registers: they run beside a whole row of scores).
__device__ __forceinline__ void tt_load8(uint32_t taddr, float* v) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tt_store8(uint32_t taddr, const float* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
                 "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])) : "memory");
}
// 128 consecutive 32-bit columns of this thread's TMEM lane.
__device__ __forceinline__ void tt_load128(uint32_t taddr, float* v) {
  uint32_t r[128];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, %80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, %96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, %112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%129];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]), "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]), "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]), "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr), "r"(taddr + 64)
      : "memory");
#pragma unroll
  for (int i = 0; i < 128; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ bool tt_no_number(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }
// 16 bytes of shared memory that another tile's warps may be writing.
__device__ __forceinline__ uint4 tt_look(const uint4* p) {
  uint4 x;
  asm volatile("ld.relaxed.cta.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(smem_u32(p)));
  return x;
}
__device__ __forceinline__ void tt_put(uint4* p, const uint32_t* w) {
  asm volatile("st.relaxed.cta.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(p)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

// DC: 64-element (128-byte) chunks of a head.
template <int DC, bool PARTS>
__global__ void __launch_bounds__(TT_THREADS, 1)
attention_tree_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TreeArgs a, int* status) {
  constexpr int D = DC * 64;
  constexpr int SUB = 128 * 128;                          // bytes of a [128 rows x 128 bytes] sub-tile
  constexpr int Q_BYTES = DC * SUB, KV_BYTES = DC * SUB, P_BYTES = 2 * SUB;
  constexpr uint32_t TMEM_COLS = 512;                     // S of both tiles: 2 x 128; O of both tiles: 2 x 128
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* q_sm = smem;                                   // 2 tiles
  uint8_t* p_sm = q_sm + 2 * Q_BYTES;                     // 2 tiles
  uint8_t* ring = p_sm + 2 * P_BYTES;                     // three buffers, in the order of use: K0 K1 V0 K2 V1 K3 V2 ...
  __shared__ uint64_t q_ready[2], full[3], empty[3], s_ready[2], s_free[2], p_ready[2], o_ready[2], apart;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag, sh_bad;
  float2 row_state = make_float2(-INFINITY, 0.f);         // keys in parts: a row's reference and sum

  pdl_trigger();
  pdl_wait();
  const int splits = PARTS ? a.splits : 1, block = blockIdx.x / splits, part = blockIdx.x - block * splits;
  const int seq = blockIdx.y / a.kv_heads, kvh = blockIdx.y - seq * a.kv_heads;
  const int q_len = min(a.seq_q_len[seq], TT_MAX_NODES), kv_len = a.seq_kv_len[seq], past = kv_len - q_len, start = a.seq_q_start[seq];
  const int group = a.heads / a.kv_heads, row0 = block * TT_ROWS, n_rows = q_len * group;
  if (row0 >= n_rows) return;                             // (the same in every block of a cluster)
  const int rows_valid = min(TT_ROWS, n_rows - row0), tiles = rows_valid > TC_BQ ? 2 : 1;
  const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.table_stride;
  // the warp's number as a value the compiler knows to be the same in every lane
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 3; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], tiles); }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_ready[t], 4);                          // one arrival per softmax warp
      mbar_init(&s_ready[t], 1);
      mbar_init(&s_free[t], 4);
      mbar_init(&p_ready[t], 4);
      mbar_init(&o_ready[t], 1);
    }
    mbar_init(&apart, 1);
    abort_flag = 0;
    sh_bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) tmem_alloc(&tmem_holder, TMEM_COLS);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_holder;
  const int page_lo = tree_low(a, past) / SB_PAGE_TOKENS, page_hi = (kv_len - 1) / SB_PAGE_TOKENS, high = tree_high(a, past, kv_len);
  int n_steps = (page_hi - page_lo) / 2 + 1, first_step = 0;
  if constexpr (PARTS) {                                  // this CTA's steps
    const int per = (n_steps + splits - 1) / splits;
    first_step = part * per;
    n_steps = max(0, min(per, n_steps - first_step));
  }
  volatile int* abort = &abort_flag;
  // A step's keys and values in the order of copies: copy n goes to buffer n % 3, whose use n / 3 it is.  The values of step i are asked for when S of step
  // i has been formed, the keys of step i + 2 when PV of step i - 1 has.  (With two buffers for the keys and one for the values a copy's whole way from
  // memory lay between PV of one step and the next.)
  auto k_copy = [&](int i) { return i == 0 ? 0 : 2 * i - 1; };
  auto v_copy = [&](int i) { return i == n_steps - 1 ? 2 * i + 1 : 2 * i + 2; };

  if (warp == 8) {
    // ---------------- producer: the whole warp walks the schedule, one elected lane issues the copies
    const bool elected = elect_one();
    int loads[3] = {0, 0, 0};                             // per buffer: how many copies were started
    for (int n = 0; n < 2 * n_steps; ++n) {
      const bool is_v = n == 2 * n_steps - 1 || (n > 0 && n % 2 == 0);
      const int i = is_v ? (n == 2 * n_steps - 1 ? n_steps - 1 : n / 2 - 1) : (n + 1) / 2, b = n % 3;
      if (n >= 3 && !__all_sync(0xffffffffu, mbar_wait(&empty[b], (n / 3 - 1) & 1, abort))) break;
      if (elected) mbar_expect_tx(&full[b], DC * SUB);
      const bool withheld = is_v && first_step + i == *(volatile int*)&tc_withhold_step;   // tests only
      for (int half = 0; half < (withheld ? 1 : 2); ++half) {
        const int row = (pages[min(page_lo + 2 * (first_step + i) + half, page_hi)] * a.kv_heads + kvh) * SB_PAGE_TOKENS;
        for (int c = 0; c < DC; ++c)
          if (elected) tma_load_2d(ring + b * KV_BYTES + c * SUB + half * 8192, is_v ? &map_v : &map_k, &full[b], c * 64, row);
      }
      loads[0] += b == 0; loads[1] += b == 1; loads[2] += b == 2;
    }
    if (*abort && elected) {                              // let the copies in flight land before the block ends
      for (int b = 0; b < 3; ++b) {
        const uint64_t begun = now_ns();
        while (loads[b] > 0 && !mbar_try(&full[b], (loads[b] - 1) & 1) && now_ns() - begun < WAIT_LIMIT_NS) {}
      }
    }
  } else if (warp == 9 || warp == 10) {
    // ---------------- MMA issuers: warp 9 for tile 0, warp 10 for tile 1, each with its own chain of waits
    const int t = warp - 9;
    if (t < tiles && n_steps > 0) {
      const bool elected = elect_one();
      const uint32_t idesc_s = instr_desc(TT_BK, 0), idesc_o = instr_desc(D, 1);
      const uint32_t q_addr = smem_u32(q_sm + t * Q_BYTES), p_addr = smem_u32(p_sm + t * P_BYTES);
      auto issue_s = [&](int buf) {
        const uint32_t k_addr = smem_u32(ring + buf * KV_BYTES);
        if (elected) {
#pragma unroll
          for (int k = 0; k < DC * 4; ++k) {
            const uint32_t off = (k >> 2) * SUB + (k & 3) * 32;
            umma_bf16(tmem_base + t * TT_BK, smem_desc(q_addr + off, 16), smem_desc(k_addr + off, 16), idesc_s,
                      k > 0 ? 1u : 0u);
          }
          umma_commit(&s_ready[t]);
          umma_commit(&empty[buf]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](bool first, int buf) {
        const uint32_t v_addr = smem_u32(ring + buf * KV_BYTES);
        if (elected) {
#pragma unroll
          for (int k = 0; k < TT_BK / 16; ++k)
            umma_bf16(tmem_base + 2 * TT_BK + t * 128, smem_desc(p_addr + (k >> 2) * SUB + (k & 3) * 32, 16),
                      smem_desc(v_addr + k * 2048, SUB), idesc_o, (first && k == 0) ? 0u : 1u);
          umma_commit(&o_ready[t]);
          umma_commit(&empty[buf]);
        }
        __syncwarp();
      };
      // every lane waits; the warp goes on together or stops together
      auto wait2 = [&](uint64_t* first_bar, uint32_t first_parity, uint64_t* second_bar, uint32_t second_parity) -> bool {
        const bool got = mbar_wait(first_bar, first_parity, abort) && mbar_wait(second_bar, second_parity, abort);
        return __all_sync(0xffffffffu, got);
      };
      bool ok = wait2(&q_ready[t], 0, &full[0], 0);
      // Tile 1 begins half a step behind tile 0: while one tile's warps wait for their scores and hand their weights over, the other's form
      // exponentials.  (In step with each other both did both at once.)
      if (ok && t == 1) ok = __all_sync(0xffffffffu, mbar_wait(&apart, 0, abort));
      if (ok) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        issue_s(0);
      }
      // Step i: S of step i+1 as soon as the softmax warps have read S of step i out of tensor memory, then PV of step i when P is written.
      for (int i = 0; i < n_steps && ok; ++i) {
        if (i + 1 < n_steps) {
          const int k = k_copy(i + 1);
          ok = wait2(&full[k % 3], (k / 3) & 1, &s_free[t], i & 1);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          issue_s(k % 3);
        }
        const int v = v_copy(i);
        ok = wait2(&full[v % 3], (v / 3) & 1, &p_ready[t], i & 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        issue_pv(i == 0, v % 3);
      }
    }
  } else if (warp < 8 && (warp >> 2) < tiles) {
    // ---------------- softmax and output: thread = packed row = tensor-memory lane.  The running output stays in tensor memory and is rescaled
    // only when a row's maximum has outgrown the reference by more than 2^8, so most steps only produce P.
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const int row = row0 + min(t * TC_BQ + r, rows_valid - 1), node = row / group;   // (rows behind the last look like the last)
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t tmem_s = tmem_base + t * TT_BK + lane_addr, tmem_o = tmem_base + 2 * TT_BK + t * 128 + lane_addr;
    uint8_t* p_row = p_sm + t * P_BYTES + r * 128;
    const int at = (start + node) * a.heads + kvh * group + row % group;   // the row's place among all heads' rows
    // Queries and results come and go 16 bytes a lane, LANES lanes a row, through shared memory (a row a lane: 32 rows a request, 2 us of 69).
    constexpr int LANES = 8 * DC;
    const int piece = lane % LANES;
    int first = 0;
    uint32_t bits[TREE_MAX_WORDS];
    {
      // K-major A operand: 64-element chunk dc, 16-byte column c ^ (r % 8) of row r
      uint8_t* q_tile = q_sm + t * Q_BYTES + (piece >> 3) * SUB;
      uint4 v[LANES];
#pragma unroll
      for (int n = 0; n < LANES; ++n) {
        const int from = __shfl_sync(0xffffffffu, at, n * (32 / LANES) + lane / LANES);
        v[n] = *reinterpret_cast<const uint4*>((const bf16*)a.q + (size_t)from * D + piece * 8);
      }
      if (a.window > 0) first = a.tok_pos[start + node] - a.window + 1;
#pragma unroll
      for (int w = 0; w < TREE_MAX_WORDS; ++w) bits[w] = tree_mask_word(a, start, node, w, q_len, first, past);
#pragma unroll
      for (int n = 0; n < LANES; ++n) {
        const int to = quarter * 32 + n * (32 / LANES) + lane / LANES;
        *reinterpret_cast<uint4*>(q_tile + to * 128 + (((piece & 7) ^ (to & 7)) << 4)) = v[n];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[t]);
    }
    float m_ref = -INFINITY, l_run = 0.f;
    bool ok = true;
    // the whole warp goes on or the whole warp stops: tensor memory is read and written by warps
    auto together = [&](bool got) -> bool { return __all_sync(0xffffffffu, got); };
    for (int i = 0; i < n_steps && ok; ++i) {
      const int j0 = (page_lo + 2 * (first_step + i)) * SB_PAGE_TOKENS;
      const bool edge = j0 + TT_BK > past || j0 < high;   // some row does not see all of the step
      ok = together(mbar_wait(&s_ready[t], i & 1, abort));
      if (!ok) break;
      if (edge) {
        // Values that are no numbers leave the tile (both tiles' warps may find the same: they write the same zeros).  The buffer's use before is over
        // (it was the keys of S above, or, for the last values, those of two steps before), so its barrier's parity speaks of this one.  Whoever finds
        // zeros where the other tile's warps found such a value has to know at the end that there was one: the flag is set in front of the zeros.
        const int n = v_copy(i);
        ok = together(mbar_wait(&full[n % 3], (n / 3) & 1, abort));
        if (!ok) break;
        uint4* v = reinterpret_cast<uint4*>(ring + n % 3 * KV_BYTES) + (warp & 3) * 32 + lane;
        constexpr int PIECES = DC * SUB / 16 / 128, FLIGHT = 4;
#pragma unroll 1
        for (int i0 = 0; i0 < PIECES; i0 += FLIGHT) {
          uint4 x[FLIGHT];
#pragma unroll
          for (int u = 0; u < FLIGHT; ++u) x[u] = tt_look(v + (i0 + u) * 128);
          bool here = false;
#pragma unroll
          for (int u = 0; u < FLIGHT; ++u)
            here |= tt_no_number(x[u].x) | tt_no_number(x[u].x >> 16) | tt_no_number(x[u].y) | tt_no_number(x[u].y >> 16) | tt_no_number(x[u].z) |
                    tt_no_number(x[u].z >> 16) | tt_no_number(x[u].w) | tt_no_number(x[u].w >> 16);
          if (here) {
            *(volatile int*)&sh_bad = 1;
            __threadfence_block();
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) {
              uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (tt_no_number(w[e])) w[e] &= 0xffff0000u;
                if (tt_no_number(w[e] >> 16)) w[e] &= 0xffffu;
              }
              tt_put(v + (i0 + u) * 128, w);
            }
          }
        }
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // The whole row of S first, so that S of the next step can be formed while the exponentials of this one run.
      float sv[128];
      tt_load128(tmem_s, sv);
      if (edge) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint64_t view = tt_view(bits, first, past, q_len, j0 + h * 64);
          const uint32_t lo = (uint32_t)view, hi = (uint32_t)(view >> 32);
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (!((e < 32 ? lo >> e : hi >> (e - 32)) & 1u)) sv[h * 64 + e] = -INFINITY;
        }
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 128; e += 8)
#pragma unroll
        for (int f = 0; f < 4; ++f) m4[f] = fmaxf(fmaxf(m4[f], sv[e + f]), sv[e + f + 4]);
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2;   // scale_log2 > 0: the maximum commutes with it
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      const bool outgrown = __any_sync(0xffffffffu, mx > m_ref + 8.f);   // also the first keys a row sees (m_ref = -inf)
      if (lane == 0) mbar_arrive(&s_free[t]);             // S of this step may be overwritten
      if (i == 0 && threadIdx.x == 0) mbar_arrive(&apart);
      if (outgrown) {
        // a new reference: rescale what has been accumulated
        const float m_new = fmaxf(m_ref, mx);
        const float alpha = m_ref == -INFINITY ? 1.f : fast_exp2(m_ref - m_new);
        if (i > 0) {
          ok = together(mbar_wait(&o_ready[t], (i - 1) & 1, abort));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
          for (int c = 0; c < D; c += 8) {
            float ov[8];
            tt_load8(tmem_o + c, ov);
#pragma unroll
            for (int e = 0; e < 8; ++e) ov[e] *= alpha;
            tt_store8(tmem_o + c, ov);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        l_run *= alpha;
        m_ref = m_new;
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
      float rs = 0.f, rs_hi = 0.f;                        // the row sum in two halves (packed adds)
      // P = exp2(S * scale - m) of 8 keys, rounded to bfloat16: one 16-byte column of the A operand
      auto exp8 = [&](int c, uint32_t* w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x0, x1;
          fma2(x0, x1, sv[c * 8 + 2 * e], sv[c * 8 + 2 * e + 1], a.scale_log2, -m_use);
          const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
          add2(rs, rs_hi, p0, p1);
          const __nv_bfloat162 two = __floats2bfloat162_rn(p0, p1);
          w[e] = *reinterpret_cast<const uint32_t*>(&two);
        }
      };
      auto store8 = [&](int c, const uint32_t* w) {
        *reinterpret_cast<uint4*>(p_row + (c >> 3) * SUB + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      };
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 8; ++c) exp8(c, pk + 4 * c);
      // P's tile is free once PV of the step before has finished
      if (i > 0 && !outgrown) ok = together(mbar_wait(&o_ready[t], (i - 1) & 1, abort));
      if (!ok) break;
#pragma unroll
      for (int c = 0; c < 8; ++c) store8(c, pk + 4 * c);
#pragma unroll
      for (int c = 8; c < 16; ++c) {
        uint32_t w[4];
        exp8(c, w);
        store8(c, w);
      }
      l_run += rs + rs_hi;
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t]);
    }
    // The tile's warps meet, also those that gave up: what one of them has found all know.
    __threadfence_block();
    __syncwarp();
    if (t) asm volatile("bar.sync 2, 128;" ::: "memory");
    else asm volatile("bar.sync 1, 128;" ::: "memory");
    if (ok && n_steps > 0) ok = together(mbar_wait(&o_ready[t], (n_steps - 1) & 1, abort));
    if (ok && n_steps > 0) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const bool bad = *(volatile int*)&sh_bad != 0;
      if constexpr (PARTS) row_state = make_float2(m_ref, l_run);
      const float inv = l_run > 0.f ? 1.f / l_run : l_run == 0.f ? 0.f : l_run;
      uint8_t* o_row = p_sm + t * P_BYTES + r * (D * 2);   // the results pass through the weights' place
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float ov[32];
        tmem_load32(tmem_o + c, ov);
        if (bad) {                                        // what was taken out of the tiles, to the rows that see it
          const int last = min((page_lo + 2 * (first_step + n_steps)) * SB_PAGE_TOKENS, kv_len);
          for (int j = (page_lo + 2 * first_step) * SB_PAGE_TOKENS; j < last; ++j) {
            if (!(tt_view(bits, first, past, q_len, j) & 1ull)) continue;
            const bf16* v = (const bf16*)a.v_store + page_row(pages[j / SB_PAGE_TOKENS], kvh, j % SB_PAGE_TOKENS, a.kv_heads, D) + c;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float x = __bfloat162float(v[e]);
              if (!(fabsf(x) < INFINITY)) ov[e] += x;
            }
          }
        }
        if constexpr (PARTS) {
#pragma unroll
          for (int d = 0; d < 32; d += 4)
            *reinterpret_cast<float4*>(part_piece<64, D>(p_sm + t * P_BYTES, q_sm + t * Q_BYTES, r, (c + d) / 4)) =
                make_float4(ov[d], ov[d + 1], ov[d + 2], ov[d + 3]);
        } else {
#pragma unroll
          for (int d = 0; d < 32; d += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 two = __floats2bfloat162_rn(ov[d + 2 * e] * inv, ov[d + 2 * e + 1] * inv);
              w[e] = *reinterpret_cast<const uint32_t*>(&two);
            }
            *reinterpret_cast<uint4*>(o_row + ((((c + d) / 8) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if constexpr (!PARTS) {
        __syncwarp();
#pragma unroll
        for (int n = 0; n < LANES; ++n) {
          const int from = n * (32 / LANES) + lane / LANES, to = __shfl_sync(0xffffffffu, at, from);
          const uint4 v = *reinterpret_cast<const uint4*>(o_row + (from - lane) * (D * 2) + ((piece ^ (from & 7)) << 4));
          if (t * TC_BQ + quarter * 32 + from < rows_valid) *reinterpret_cast<uint4*>((bf16*)a.out + (size_t)to * D + piece * 8) = v;
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if constexpr (PARTS) {
    // (the rows' states lie where keys were: both tiles are done with them behind the block's barrier)
    float2* ml = reinterpret_cast<float2*>(ring);
    __syncthreads();
    if (threadIdx.x < TT_ROWS) ml[threadIdx.x] = row_state;
    cluster_barrier();
    // every CTA joins its share of the rows: 16 threads a row, D / 16 columns each
    constexpr int COLS = D / 16;
    const int share = (rows_valid + splits - 1) / splits, c = (threadIdx.x & 15) * COLS;
    if (threadIdx.x < TT_ROWS) {
      for (int n = threadIdx.x >> 4; n < share; n += TT_ROWS / 16) {
        const int mine = part * share + n;
        if (mine >= rows_valid) break;
        const int t = mine / TC_BQ, r = mine % TC_BQ;
        // (all loads in front of what they decide: a part without keys filed nothing, and what is read there is not used)
        float2 ps[TT_MAX_SPLITS];
        float4 x[TT_MAX_SPLITS][COLS / 4];
        float top = -INFINITY, sum = 0.f, o[COLS];
#pragma unroll
        for (int p = 0; p < TT_MAX_SPLITS; ++p) {
          ps[p] = make_float2(-INFINITY, 0.f);
          if (p >= splits) continue;
          ps[p] = peer_load2(peer_u32(ml + mine, p));
#pragma unroll
          for (int d = 0; d < COLS / 4; ++d)
            x[p][d] = peer_load4(peer_u32(part_piece<64, D>(p_sm + t * P_BYTES, q_sm + t * Q_BYTES, r, c / 4 + d), p));
        }
#pragma unroll
        for (int p = 0; p < TT_MAX_SPLITS; ++p)
          if (ps[p].y != 0.f) top = fmaxf(top, ps[p].x);
#pragma unroll
        for (int d = 0; d < COLS; ++d) o[d] = 0.f;
#pragma unroll
        for (int p = 0; p < TT_MAX_SPLITS; ++p) {
          // (a part whose sum is no number has a score that is none, which is the row's result)
          if (p >= splits || ps[p].y == 0.f) continue;
          const float w = fast_exp2(ps[p].x - top);
          sum = fmaf(w, ps[p].y, sum);
#pragma unroll
          for (int d = 0; d < COLS / 4; ++d) {
            o[4 * d] = fmaf(w, x[p][d].x, o[4 * d]); o[4 * d + 1] = fmaf(w, x[p][d].y, o[4 * d + 1]);
            o[4 * d + 2] = fmaf(w, x[p][d].z, o[4 * d + 2]); o[4 * d + 3] = fmaf(w, x[p][d].w, o[4 * d + 3]);
          }
        }
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
        const int row = row0 + mine;
        bf16* dst = (bf16*)a.out + ((size_t)(start + row / group) * a.heads + kvh * group + row % group) * D + c;
#pragma unroll
        for (int d = 0; d < COLS; d += 4) {
          const __nv_bfloat162 two = __floats2bfloat162_rn(o[d] * inv, o[d + 1] * inv), more = __floats2bfloat162_rn(o[d + 2] * inv, o[d + 3] * inv);
          *reinterpret_cast<uint2*>(dst + d) = make_uint2(*reinterpret_cast<const uint32_t*>(&two), *reinterpret_cast<const uint32_t*>(&more));
        }
      }
    }
    tree_cluster_leave();
  }
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tmem_free(tmem_holder, TMEM_COLS);
  }
  if (threadIdx.x == 0 && abort_flag && status) atomicOr(status, 16);
}

// ------------------------------------------------------------------------------------------ host

template <int DC> static constexpr int tt_smem() { return (2 * DC + 4 + 3 * DC) * 128 * 128 + 1024; }

template <int DC, bool PARTS>
static int launch_as(const CUtensorMap& mk, const CUtensorMap& mv, const TreeArgs& a, int seqs, int max_q_len, int* status, cudaStream_t s) {
  const int e = allow_smem<&attention_tree_tc_kernel<DC, PARTS>>(tt_smem<DC>());
  if (e) return e;
  const int blocks = (max_q_len * (a.heads / a.kv_heads) + TT_ROWS - 1) / TT_ROWS;
  const dim3 grid(blocks * a.splits, seqs * a.kv_heads);
  if (PARTS) return launch_dependent_cluster(attention_tree_tc_kernel<DC, PARTS>, grid, dim3(TT_THREADS), tt_smem<DC>(), s, dim3(a.splits), mk, mv, a, status);
  return launch_dependent(attention_tree_tc_kernel<DC, PARTS>, grid, dim3(TT_THREADS), tt_smem<DC>(), s, mk, mv, a, status);
}

static unsigned long long next_limit_ns = WAIT_LIMIT_NS;
static int next_withhold_step = -1;

extern "C" {

// For tests of the give-up path: the NEXT sb_attention_tree_tc launch leaves out half of the values of step `step` (128 keys) of every block
// and its waits give up after `limit_ns`.  The blocks cannot finish; the launch must return with bit 16 of *status set.
void sb_attention_tree_tc_withhold(int step, unsigned long long limit_ns) {
  next_withhold_step = step;
  next_limit_ns = limit_ns ? limit_ns : WAIT_LIMIT_NS;
}

// How many clusters of `size` of its CTAs, which take an SM each, the current device runs at once, or minus an error.
int sb_attention_tree_tc_clusters(int size) {
  auto kernel = attention_tree_tc_kernel<2, true>;
  const int set = allow_smem<&attention_tree_tc_kernel<2, true>>(tt_smem<2>());
  if (set) return -set;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(TT_THREADS);
  cfg.dynamicSmemBytes = tt_smem<2>();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
  return e == cudaSuccess ? n : -(int)e;
}

// bfloat16, dim 64 or 128 (-2 otherwise), scale > 0, q, out and the stores 16-byte aligned; splits 1, 2, 4 or 8; n_pages: pages in the stores.
int sb_attention_tree_tc(const void* q, void* out, const void* k_store, const void* v_store, int n_pages, const int* block_table,
                         int table_stride, const int* seq_slot, const int* seq_q_start, const int* seq_q_len, const int* seq_kv_len,
                         const int* tok_pos, const void* mask, int words, int seqs, int max_q_len, int heads, int kv_heads, int dim,
                         float scale, int window, int splits, int* status, cudaStream_t s) {
  if (seqs == 0 || max_q_len == 0) return 0;
  if (kv_heads <= 0 || heads % kv_heads || words < 1 || !(scale > 0.f) || max_q_len > TT_MAX_NODES) return -2;
  if ((dim != 64 && dim != 128) || (splits != 1 && splits != 2 && splits != 4 && splits != TT_MAX_SPLITS)) return -2;
  if ((long long)seqs * kv_heads > 65535) return -2;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_store | (uintptr_t)v_store) & 15) return -2;
  // (a TMA coordinate is 32 bits)
  const long long kv_rows = (long long)n_pages * kv_heads * SB_PAGE_TOKENS;
  if (kv_rows > 0x7fffffffll) return -2;
  CUtensorMap mk, mv;
  int rc = sb_make_map(&mk, k_store, kv_rows, dim, SB_PAGE_TOKENS);
  if (rc) return rc;
  rc = sb_make_map(&mv, v_store, kv_rows, dim, SB_PAGE_TOKENS);
  if (rc) return rc;
  const TreeArgs a{q, out, k_store, v_store, block_table, table_stride, seq_slot, seq_q_start, seq_q_len, seq_kv_len, tok_pos,
                   (const uint32_t*)mask, words, words < TREE_MAX_WORDS ? words : TREE_MAX_WORDS, heads, kv_heads, dim,
                   scale * 1.4426950408889634f, window > 0 ? window : 0, splits};
  const bool test_run = next_withhold_step >= 0;
  if (test_run) {
    cudaMemcpyToSymbolAsync(tc_withhold_step, &next_withhold_step, sizeof(int), 0, cudaMemcpyHostToDevice, s);
    cudaMemcpyToSymbolAsync(tc_wait_limit_ns, &next_limit_ns, sizeof(next_limit_ns), 0, cudaMemcpyHostToDevice, s);
    cudaStreamSynchronize(s);
  }
  if (dim == 64) rc = splits > 1 ? launch_as<1, true>(mk, mv, a, seqs, max_q_len, status, s) : launch_as<1, false>(mk, mv, a, seqs, max_q_len, status, s);
  else rc = splits > 1 ? launch_as<2, true>(mk, mv, a, seqs, max_q_len, status, s) : launch_as<2, false>(mk, mv, a, seqs, max_q_len, status, s);
  if (test_run) {
    cudaStreamSynchronize(s);
    next_withhold_step = -1;
    next_limit_ns = WAIT_LIMIT_NS;
    cudaMemcpyToSymbolAsync(tc_withhold_step, &next_withhold_step, sizeof(int), 0, cudaMemcpyHostToDevice, s);
    cudaMemcpyToSymbolAsync(tc_wait_limit_ns, &next_limit_ns, sizeof(next_limit_ns), 0, cudaMemcpyHostToDevice, s);
    cudaStreamSynchronize(s);
  }
  return rc;
}

}  // extern "C"
