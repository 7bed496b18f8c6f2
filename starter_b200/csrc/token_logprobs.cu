// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits, in one pass over them.
//
// With m a row's largest entry, L = sum exp(x_i - m) and T = sum exp(x_i - m) (x_i - m):
//     lse = m + log L,   log p(t) = (x_t - m) - log L,   H = log L - T / L.
// Every thread keeps (m, L, T) of what it has seen, all float; a new reference m' scales L by a = exp(m - m') and makes
// T a (T + L (m - m')).  Entries of minus infinity add nothing to any of them.  The alternatives are the largest entries, the lowest
// index first among equals: a warp keeps the best 32 it has seen, sorted, one to a lane, and looks closer only at tiles whose largest
// entry beats its k-th (or is not worse than the best k-th any warp of the block has: k entries above it are known then).  Entries that
// are no numbers are never listed.
//
// A row is shared by the blocks of a cluster, whose results meet in the first one's hands.  What bounds it is reading the logits.
#include "logprob_stats.cuh"

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_MAX_TOP 32
#define LP_MAX_CLUSTER 8
#define LP_NONE 0x7fffffff

struct Item { float v; int i; };
__device__ __forceinline__ bool lp_before(const Item& a, const Item& b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
__device__ __forceinline__ Item lp_shfl(const Item& a, int lane) {
  return Item{__shfl_sync(0xffffffffu, a.v, lane), __shfl_sync(0xffffffffu, a.i, lane)};
}
// The best 32 of two sorted lists (best in lane 0): the other one backwards against this one leaves them as a bitonic sequence.
__device__ __forceinline__ Item lp_merge(Item a, const Item& b_lane) {
  const int lane = threadIdx.x & 31;
  const Item b = lp_shfl(b_lane, 31 - lane);
  if (lp_before(b, a)) a = b;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Item other{__shfl_xor_sync(0xffffffffu, a.v, o), __shfl_xor_sync(0xffffffffu, a.i, o)};
    if (lp_before(other, a) == ((lane & o) == 0)) a = other;
  }
  return a;
}

struct LogprobArgs {
  const void* logits;
  long long row_stride;       // entries
  int vocab, top;
  const int* tokens;          // [rows]; negative: none (its log probability is 0)
  float* given;               // [rows]
  float* entropy;             // [rows]
  float* top_value;           // [rows, top]
  int* top_id;
  int* status;
};

__device__ __forceinline__ uint32_t lp_peer(const void* p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float lp_peer_load(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ void lp_cluster_barrier() {
  __syncwarp();                    // (.aligned: a whole warp at once)
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS) token_logprobs_kernel(const LogprobArgs a, int parts) {
  constexpr int VEC = 16 / sizeof(T), U = 16 / VEC;       // entries of a 16-byte load; loads a thread has on their way
  constexpr int N = VEC * U;
  __shared__ float sh_stats[LP_WARPS][3], cl_stats[3];
  __shared__ float sh_v[LP_WARPS][32], cl_v[32];
  __shared__ int sh_i[LP_WARPS][32], cl_i[32];
  __shared__ float sh_floor;                              // the best k-th entry any warp has
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.y, part = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = (const T*)a.logits + (size_t)row * a.row_stride;
  // loads start on 16-byte boundaries: the row is `off` entries behind one
  const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
  const T* aligned = x - off;
  if (threadIdx.x == 0) sh_floor = -INFINITY;
  __syncthreads();

  const long long vectors = ((long long)off + a.vocab + VEC - 1) / VEC;
  const int per_tile = LP_THREADS * U;
  const int tiles = (int)((vectors + per_tile - 1) / per_tile);
  Stats st{-INFINITY, 0.f, 0.f};
  Item best{-INFINITY, LP_NONE}, kth{-INFINITY, LP_NONE};
  uint4 raw[U];
  auto load = [&](int tile) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long first = ((long long)tile * per_tile + u * LP_THREADS + threadIdx.x) * VEC - off;    // of the row
      if (first >= 0 && first + VEC <= a.vocab) {
        raw[u] = __ldcs(reinterpret_cast<const uint4*>(x + first));
      } else {                                            // the row's ends, entry by entry; minus infinity beside them
        T e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = first + i >= 0 && first + i < a.vocab ? x[first + i] : from_f<T>(-INFINITY);
        raw[u] = *reinterpret_cast<uint4*>(e);
      }
    }
  };
  if (part < tiles) load(part);
  for (int tile = part; tile < tiles; tile += parts) {
    float v[N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          v[u * VEC + i] = __uint_as_float(w[i]);
        } else {
          v[u * VEC + 2 * i] = __uint_as_float(w[i] << 16);
          v[u * VEC + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
    if (tile + parts < tiles) load(tile + parts);
    float mx = v[0];
#pragma unroll
    for (int e = 1; e < N; ++e) mx = fmaxf(mx, v[e]);
    if (mx > st.m) {
      const Stats here{mx, 0.f, 0.f};
      st = lp_join(st, here);
    }
    const float base = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = v[e] - base, p = lp_exp(d);
      st.l += p;
      st.t = fmaf(p, fmaxf(d, -1e30f), st.t);
    }
    if constexpr (TOP) {
      const float floor = *(volatile float*)&sh_floor;
      if (__any_sync(0xffffffffu, (mx > kth.v || kth.i == LP_NONE) && mx >= floor)) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const long long place = ((long long)tile * per_tile + (e / VEC) * LP_THREADS + threadIdx.x) * VEC + e % VEC - off;
          const Item mine{v[e], place >= 0 && place < a.vocab ? (int)place : LP_NONE};
          uint32_t left = __ballot_sync(0xffffffffu, lp_before(mine, kth) && mine.v >= floor);
          while (left) {
            const Item cand = lp_shfl(mine, __ffs(left) - 1);
            left &= left - 1;
            if (!lp_before(cand, kth)) continue;          // (the same in every lane)
            const int at = __popc(__ballot_sync(0xffffffffu, lp_before(best, cand)));
            const Item up{__shfl_up_sync(0xffffffffu, best.v, 1), __shfl_up_sync(0xffffffffu, best.i, 1)};
            if (lane == at) best = cand;
            else if (lane > at) best = up;
            kth = lp_shfl(best, a.top - 1);
          }
        }
        if (lane == 0 && kth.i != LP_NONE && kth.v > floor) *(volatile float*)&sh_floor = kth.v;   // (any warp's is true; a lost race costs a look)
      }
    }
  }

  // the lanes', then the warps', then the blocks' parts
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stats other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.l, o), __shfl_xor_sync(0xffffffffu, st.t, o)};
    st = lp_join(st, other);
  }
  if (lane == 0) { sh_stats[warp][0] = st.m; sh_stats[warp][1] = st.l; sh_stats[warp][2] = st.t; }
  if (TOP) { sh_v[warp][lane] = best.v; sh_i[warp][lane] = best.i; }
  __syncthreads();
  auto fold = [&]() {                                     // the lists of sh_v, sh_i into warp 0's registers
    for (int half = LP_WARPS / 2; half > 0; half >>= 1) {
      if (warp < half) {
        best = lp_merge(best, Item{sh_v[warp + half][lane], sh_i[warp + half][lane]});
        sh_v[warp][lane] = best.v;
        sh_i[warp][lane] = best.i;
      }
      __syncthreads();
    }
  };
  if (TOP) fold();
  if (warp == 0) {
    st = lane < LP_WARPS ? Stats{sh_stats[lane][0], sh_stats[lane][1], sh_stats[lane][2]} : Stats{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Stats other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.l, o), __shfl_xor_sync(0xffffffffu, st.t, o)};
      st = lp_join(st, other);
    }
  }
  if (parts > 1) {
    if (warp == 0) {
      if (lane == 0) { cl_stats[0] = st.m; cl_stats[1] = st.l; cl_stats[2] = st.t; }
      if (TOP) { cl_v[lane] = best.v; cl_i[lane] = best.i; }
    }
    __syncthreads();
    lp_cluster_barrier();
    if (part == 0) {
      if (TOP) {
        best = Item{-INFINITY, LP_NONE};
        if (warp < parts) {
          best.v = lp_peer_load(lp_peer(&cl_v[lane], warp));
          best.i = __float_as_int(lp_peer_load(lp_peer(&cl_i[lane], warp)));
        }
        sh_v[warp][lane] = best.v;
        sh_i[warp][lane] = best.i;
        __syncthreads();
        fold();
      }
      if (warp == 0) {
        st = Stats{-INFINITY, 0.f, 0.f};
        if (lane < parts)
          st = Stats{lp_peer_load(lp_peer(&cl_stats[0], lane)), lp_peer_load(lp_peer(&cl_stats[1], lane)), lp_peer_load(lp_peer(&cl_stats[2], lane))};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const Stats other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.l, o), __shfl_xor_sync(0xffffffffu, st.t, o)};
          st = lp_join(st, other);
        }
      }
    }
    lp_cluster_barrier();                                 // nobody leaves while it is read
    if (part) return;
  }
  if (warp == 0) {
    // (a sum that is no number, or of nothing, makes a row whose probabilities are none)
    const float log_l = st.l > 0.f ? logf(st.l) : NAN;
    if (lane == 0) {
      const int t = a.tokens[row];
      float given = 0.f;
      if (t >= a.vocab) {
        given = NAN;
        if (a.status) atomicOr(a.status, 1);
      } else if (t >= 0) {
        given = (to_f<T>(x[t]) - st.m) - log_l;
      }
      a.given[row] = given;
      a.entropy[row] = log_l - st.t / st.l;
    }
    if (TOP && lane < a.top) {
      a.top_value[(size_t)row * a.top + lane] = (best.v - st.m) - log_l;
      a.top_id[(size_t)row * a.top + lane] = best.i == LP_NONE ? -1 : best.i;
    }
  }
}

template <typename T, bool TOP>
static int launch_rows(const LogprobArgs& a, int rows, int parts, cudaStream_t s) {
  for (int first = 0; first < rows; first += 65535) {     // (a grid's dimension)
    LogprobArgs b = a;
    const int here = rows - first < 65535 ? rows - first : 65535;
    b.logits = (const T*)a.logits + (size_t)first * a.row_stride;
    b.tokens += first; b.given += first; b.entropy += first;
    if (TOP) { b.top_value += (size_t)first * a.top; b.top_id += (size_t)first * a.top; }
    const int rc = launch_dependent_cluster(token_logprobs_kernel<T, TOP>, dim3(parts, here), dim3(LP_THREADS), 0, s, dim3(parts), b, parts);
    if (rc) return rc;
  }
  return 0;
}

extern "C" {

int sb_token_logprobs_max_top() { return LP_MAX_TOP; }

// logits: [rows, vocab], dtype 0 float, 1 bfloat16, rows `row_stride` entries apart; tokens [rows]; top 0 to 32, at most vocab;
// given, entropy [rows]; top_value, top_id [rows, top] (null with top 0); parts: 1, 2, 4 or 8 blocks a row.  A token of vocab or more sets
// bit 1 of *status (null: not told) and has no log probability.
int sb_token_logprobs(int dtype, const void* logits, int rows, int vocab, long long row_stride, const int* tokens, int top, float* given,
                      float* entropy, float* top_value, int* top_id, int parts, int* status, cudaStream_t s) {
  if (rows == 0) return 0;
  if (vocab < 1 || top < 0 || top > LP_MAX_TOP || top > vocab || row_stride < 0) return -2;
  if (parts != 1 && parts != 2 && parts != 4 && parts != LP_MAX_CLUSTER) return -2;
  if (vocab > 0x7fffff00 || ((uintptr_t)logits & (dtype == 0 ? 3 : 1))) return -2;
  const LogprobArgs a{logits, row_stride, vocab, top, tokens, given, entropy, top_value, top_id, status};
  if (dtype == 0) return top ? launch_rows<float, true>(a, rows, parts, s) : launch_rows<float, false>(a, rows, parts, s);
  if (dtype == 1) return top ? launch_rows<bf16, true>(a, rows, parts, s) : launch_rows<bf16, false>(a, rows, parts, s);
  return -1;
}

}  // extern "C"
