// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits, in one pass over them.
//
// With m a row's largest entry, L = sum exp(x_i - m) and T = sum exp(x_i - m) (x_i - m):
//     lse = m + log L,   log p(t) = (x_t - m) - log L,   H = log L - T / L.
// Every thread keeps (m, L, T) of what it has seen, all float; a new reference m' scales L by a = exp(m - m') and makes
// T a (T + L (m - m')).  Entries of minus infinity add nothing to any of them.
//
// The alternatives are the k largest entries, the lowest index first among equals.  The pass itself leaves only the largest entry of every 64
// bytes of the row in shared memory: of such groups, ordered by their largest entry and then by place, the first k hold all alternatives
// (an entry of another group has k entries in front of it).  Behind the pass the block finds those groups and reads them once more: a bar that k + 1
// of them reach comes from the threads' best ones, what reaches it is ranked by counting, and so are the groups' entries.  A value and
// an index make one 64-bit key, larger for what comes first, so that all keys differ.  (Candidates gathered in the pass itself, into a sorted
// list a warp or a buffer a block, cost barriers and divergent code in every tile: 8 rows of 151,936 with 20 alternatives 30 and 17 us, 8.5 so; 600
// rows with 5 110 and 138, 66 so.)  Entries that are no numbers have no key.
//
// A row is shared by the blocks of a cluster, whose results meet in the first one's hands.  What bounds it is reading the logits where rows are many
// (600 of 151,936 in float, 365 MB: 5.5 TB/s); of the 8.5 us of 8 rows the pass takes 2, the choice of the alternatives 3.5, the meeting 2.
// In bfloat16 the same rows take 42.6 us where the bytes are worth 28: the exponentials, 20 us of the special-function unit, do not hide behind loads a
// tile ahead (two entries at once in the other operations: 44.3 before).  Two or three tiles ahead cost blocks an SM: 64 rows 28 us against 17.
#include "allow_smem.cuh"
#include "logprob_stats.cuh"

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_MAX_TOP 32
#define LP_MAX_CLUSTER 8
#define LP_BYTES 64                      // a thread's piece of a tile: a group
#define LP_TILE_BYTES (LP_THREADS * LP_BYTES)
#define LP_QUADS (LP_THREADS / 4)
#define LP_BUFFER 1088                   // keys: the entries of LP_MAX_TOP + 1 groups, and a cluster's lists
#define LP_MAX_SLOTS 160                 // tiles of a block whose groups' largest entries shared memory holds

typedef unsigned long long Key;
// 0: none.  (Both zeros are one value.)
__device__ __forceinline__ Key lp_key(float v, int i) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return v == v ? (Key)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i : 0ull;
}
__device__ __forceinline__ float lp_value(Key k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
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
__device__ __forceinline__ Key lp_peer_key(uint32_t a) {
  Key v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void lp_cluster_arrive() {
  __syncwarp();                    // (.aligned: a whole warp at once)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void lp_cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The parts of `lanes` lanes, a power of two, joined: in every one of them.
__device__ __forceinline__ void lp_join_lanes(Stats& st, int lanes) {
#pragma unroll
  for (int o = lanes / 2; o > 0; o >>= 1) {
    const Stats other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.l, o), __shfl_xor_sync(0xffffffffu, st.t, o)};
    st = lp_join(st, other);
  }
}

// Two floats at once.
__device__ __forceinline__ Key lp_two(float a, float b) {
  Key r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 lp_apart(Key k) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(k));
  return r;
}
__device__ __forceinline__ Key lp_add2(Key a, Key b) {
  Key r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Key lp_mul2(Key a, Key b) {
  Key r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Key lp_fma2(Key a, Key b, Key c) {
  Key r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 32 bytes on their boundary, which are not needed again.
__device__ __forceinline__ void lp_load32(uint32_t* w, const void* p) {
  asm volatile("ld.global.cs.v4.b64 {%0, %1, %2, %3}, [%4];"
               : "=l"(reinterpret_cast<Key*>(w)[0]), "=l"(reinterpret_cast<Key*>(w)[1]), "=l"(reinterpret_cast<Key*>(w)[2]), "=l"(reinterpret_cast<Key*>(w)[3])
               : "l"(p));
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 4) token_logprobs_kernel(const LogprobArgs a, int rest) {
  constexpr int N = LP_BYTES / sizeof(T), HALF = N / 2;   // entries of a thread's piece, in two loads
  extern __shared__ float maxima[];                       // [tiles of this block][LP_THREADS]
  __shared__ float sh_stats[LP_WARPS][3], cl_stats[3];
  __shared__ Key buffer[TOP ? LP_BUFFER : 1], list[LP_MAX_TOP + 1], quad_best[LP_QUADS], sh_bar;
  __shared__ int sh_count;
  // A launch whose rows are the rest of the one directly in front of it (`rest`) reads the logits while that one still runs: its blocks are there
  // once every block of the other has passed its own wait, which the logits were complete for.  It waits in front of its first write.
  if (!rest) pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y, parts = gridDim.x, part = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = (const T*)a.logits + (size_t)row * a.row_stride;
  // loads start on 32-byte boundaries: the row is `off` entries behind one
  const int off = (int)(((uintptr_t)x & 31) / sizeof(T));
  const int tiles = (int)(((long long)off + a.vocab + LP_THREADS * N - 1) / (LP_THREADS * N));
  const int slots = part < tiles ? (tiles - part + parts - 1) / parts : 0;
  auto first_of = [&](int slot, int thread) -> long long {   // the first entry of a thread's piece of a tile
    return ((long long)(part + slot * parts) * LP_THREADS + thread) * N - off;
  };
  Stats st{-INFINITY, 0.f, 0.f};
  int best_slot = -1;                                     // the tile of the thread's largest entry
  uint32_t raw[LP_BYTES / 4];
  auto load = [&](int slot) {
    const long long first = first_of(slot, threadIdx.x);
    if (first >= 0 && first + N <= a.vocab) {
      lp_load32(raw, x + first);
      lp_load32(raw + LP_BYTES / 8, x + first + HALF);
    } else {                                              // the row's ends, entry by entry; minus infinity beside them
#pragma unroll
      for (int w = 0; w < LP_BYTES / 4; ++w) {
        if constexpr (sizeof(T) == 4) {
          raw[w] = first + w >= 0 && first + w < a.vocab ? reinterpret_cast<const uint32_t*>(x)[first + w] : 0xff800000u;
        } else {
          const long long e = first + 2 * w;
          const uint32_t lo = e >= 0 && e < a.vocab ? reinterpret_cast<const uint16_t*>(x)[e] : 0xff80u;
          const uint32_t hi = e + 1 >= 0 && e + 1 < a.vocab ? reinterpret_cast<const uint16_t*>(x)[e + 1] : 0xff80u;
          raw[w] = lo | hi << 16;
        }
      }
    }
  };
  int slot = slots ? row * 11 % slots : 0;
  if (slots) load(slot);
  for (int n = 0; n < slots; ++n) {
    const int next = slot + 1 < slots ? slot + 1 : 0;
    float v[N];
#pragma unroll
    for (int w = 0; w < LP_BYTES / 4; ++w) {
      if constexpr (sizeof(T) == 4) {
        v[w] = __uint_as_float(raw[w]);
      } else {
        v[2 * w] = __uint_as_float(raw[w] << 16);
        v[2 * w + 1] = __uint_as_float(raw[w] & 0xffff0000u);
      }
    }
    if (n + 1 < slots) load(next);
    float mx = v[0];
#pragma unroll
    for (int e = 1; e < N; ++e) mx = fmaxf(mx, v[e]);
    if (TOP) maxima[slot * LP_THREADS + threadIdx.x] = mx;
    if (mx > st.m) {
      st = lp_join(st, Stats{mx, 0.f, 0.f});
      best_slot = slot;
    }
    const float base = st.m == -INFINITY ? 0.f : st.m;
    const Key from = lp_two(-base, -base), log2e = lp_two(1.4426950408889634f, 1.4426950408889634f);
    Key l = lp_two(st.l, 0.f), t = lp_two(st.t, 0.f);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const Key d = lp_add2(lp_two(v[e], v[e + 1]), from);
      const float2 far = lp_apart(d), power = lp_apart(lp_mul2(d, log2e));
      const Key p = lp_two(lp_exp2(power.x), lp_exp2(power.y));
      l = lp_add2(l, p);
      t = lp_fma2(p, lp_two(fmaxf(far.x, -1e30f), fmaxf(far.y, -1e30f)), t);
    }
    const float2 ls = lp_apart(l), ts = lp_apart(t);
    st.l = ls.x + ls.y;
    st.t = ts.x + ts.y;
    slot = next;
  }

  // The `want` best of the buffer's `count` keys to list, in order (zeros behind them); four lanes count for a key.  Every thread, between barriers.
  const int quad = threadIdx.x / 4, in_quad = threadIdx.x & 3;
  auto over_quad = [&](int n) { n += __shfl_xor_sync(0xffffffffu, n, 1); return n + __shfl_xor_sync(0xffffffffu, n, 2); };
  auto rank = [&](int count, int want) {
    if (threadIdx.x <= LP_MAX_TOP) list[threadIdx.x] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < count; i0 += LP_QUADS) {
      const Key mine = i0 + quad < count ? buffer[i0 + quad] : 0;
      int above = 0;
#pragma unroll 4
      for (int j = in_quad; j < count; j += 4) above += buffer[j] > mine;
      above = over_quad(above);
      if (in_quad == 0 && mine && above < want) list[above] = mine;
    }
    __syncthreads();
  };
  if constexpr (TOP) {
    // One group more than alternatives: the row's first one may begin in front of the row, and name what stands there its best.
    const int want = a.top + 1;
    auto group_key = [&](int slot) { return lp_key(maxima[slot * LP_THREADS + threadIdx.x], slot * LP_THREADS + threadIdx.x); };
    Key best = 0;
    if (best_slot >= 0) best = lp_key(st.m, best_slot * LP_THREADS + threadIdx.x);
    else                                                  // (nothing above minus infinity)
      for (int s = 0; s < slots; ++s) best = max(best, group_key(s));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (in_quad == 0) quad_best[quad] = best;
    if (threadIdx.x == 0) sh_count = 0;
    __syncthreads();
    int better = 0;
#pragma unroll
    for (int n = 0; n < LP_QUADS / 4; ++n) {
      const int j = 4 * n + in_quad;
      better += quad_best[j] > best || (quad_best[j] == best && j < quad);
    }
    better = over_quad(better);
    if (in_quad == 0 && better == want - 1) sh_bar = best;   // `want` groups reach it (or there are not that many, and it is 0)
    __syncthreads();
    {
      const Key bar = sh_bar;
      const float value = bar ? lp_value(bar) : -INFINITY;
#pragma unroll 8
      for (int s = 0; s < slots; ++s) {
        if (!(maxima[s * LP_THREADS + threadIdx.x] >= value)) continue;
        const Key key = group_key(s);
        if (key >= bar) {
          const int at = atomicAdd(&sh_count, 1);
          if (at < LP_BUFFER) buffer[at] = key;
        }
      }
    }
    __syncthreads();
    int count = sh_count;
    if (count <= LP_BUFFER) {
      rank(count, want);
    } else {
      // (a few threads hold far more of the best groups than their share: the best of all, the best below it, and so on)
      Key last = ~0ull;
      for (int n = 0; n < want; ++n) {
        Key mine = 0;
        for (int s = 0; s < slots; ++s) {
          const Key key = group_key(s);
          if (key < last) mine = max(mine, key);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        if (lane == 0) quad_best[warp] = mine;
        __syncthreads();
        last = 0;
        for (int w = 0; w < LP_WARPS; ++w) last = max(last, quad_best[w]);
        if (threadIdx.x == 0) list[n] = last;
        __syncthreads();
      }
    }
    // the groups' entries that reach the k-th group's best
    const float bar = list[a.top - 1] ? lp_value(list[a.top - 1]) : -INFINITY;
    if (threadIdx.x == 0) sh_count = 0;
    __syncthreads();
    for (int idx = threadIdx.x; idx < want * N; idx += LP_THREADS) {
      const Key group = list[idx / N];
      if (group == 0) break;
      const int id = (int)~(uint32_t)group;
      const long long place = first_of(id / LP_THREADS, id % LP_THREADS) + idx % N;
      if (place < 0 || place >= a.vocab) continue;
      const float value = to_f<T>(x[place]);
      if (value >= bar) buffer[atomicAdd(&sh_count, 1)] = lp_key(value, (int)place);
    }
    __syncthreads();
    count = sh_count;
    rank(count, a.top);
  }

  // the lanes', then the warps', then the blocks' parts
  lp_join_lanes(st, 32);
  if (lane == 0) { sh_stats[warp][0] = st.m; sh_stats[warp][1] = st.l; sh_stats[warp][2] = st.t; }
  if (threadIdx.x == 0) sh_count = 0;
  __syncthreads();
  if (warp == 0) {
    const int w = lane % LP_WARPS;
    st = Stats{sh_stats[w][0], sh_stats[w][1], sh_stats[w][2]};
    lp_join_lanes(st, LP_WARPS);
  }
  if (parts > 1) {
    if (threadIdx.x == 0) { cl_stats[0] = st.m; cl_stats[1] = st.l; cl_stats[2] = st.t; }
    lp_cluster_arrive();
    lp_cluster_wait();
    if (part == 0) {
      if (TOP) {
        // Of the blocks' lists, each in order, what reaches the least of their n-th entries, n parts >= top: at least `top` do.
        const int n = (a.top + parts - 1) / parts - 1;
        Key mine = 0, bar = ~0ull;
        if (threadIdx.x < parts * a.top) mine = lp_peer_key(lp_peer(&list[threadIdx.x % a.top], threadIdx.x / a.top));
        for (int p = 0; p < parts; ++p) bar = min(bar, lp_peer_key(lp_peer(&list[n], p)));
        if (mine && mine >= bar) buffer[atomicAdd(&sh_count, 1)] = mine;
      }
      if (warp == 0) {
        const int p = lane % parts;
        st = Stats{lp_peer_load(lp_peer(&cl_stats[0], p)), lp_peer_load(lp_peer(&cl_stats[1], p)), lp_peer_load(lp_peer(&cl_stats[2], p))};
        lp_join_lanes(st, parts);
      }
    }
    lp_cluster_arrive();
    if (part) {
      lp_cluster_wait();                                  // nobody leaves while it is read
      return;
    }
    if (TOP) {
      __syncthreads();
      rank(sh_count, a.top);
    }
    lp_cluster_wait();
  }
  if (warp == 0) {
    if (rest) pdl_wait();
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
      const Key key = list[lane];
      a.top_value[(size_t)row * a.top + lane] = ((key ? lp_value(key) : -INFINITY) - st.m) - log_l;
      a.top_id[(size_t)row * a.top + lane] = key ? (int)~(uint32_t)key : -1;
    }
  }
}

// Tiles of a block with the most of them.
template <typename T> static int lp_slots(int vocab, int parts) {
  const long long tiles = ((long long)vocab + 31 / (int)sizeof(T) + LP_TILE_BYTES / (int)sizeof(T) - 1) / (LP_TILE_BYTES / (int)sizeof(T));
  return (int)((tiles + parts - 1) / parts);
}

template <typename T, bool TOP>
static int launch_rows(LogprobArgs a, int first, int rows, int parts, int rest, cudaStream_t s) {
  int smem = 0;
  if (TOP) {
    // (with less than the launch in front of it, an SM would have to be empty before it could divide its memory anew)
    const int slots = lp_slots<T>(a.vocab, rest ? 1 : parts);
    if (slots > LP_MAX_SLOTS) return -2;
    smem = slots * LP_THREADS * 4;
    const int e = allow_smem<&token_logprobs_kernel<T, TOP>>(smem);
    if (e) return e;
  }
  a.logits = (const T*)a.logits + (size_t)first * a.row_stride;
  a.tokens += first; a.given += first; a.entropy += first;
  if (TOP) { a.top_value += (size_t)first * a.top; a.top_id += (size_t)first * a.top; }
  while (rows > 0) {                                      // (a grid's dimension counts 65,535 rows)
    const int here = rows < 65535 ? rows : 65535;
    const int rc = launch_dependent_cluster(token_logprobs_kernel<T, TOP>, dim3(parts, here), dim3(LP_THREADS), smem, s, dim3(parts), a, rest);
    if (rc) return rc;
    a.logits = (const T*)a.logits + (size_t)here * a.row_stride;
    a.tokens += here; a.given += here; a.entropy += here;
    if (TOP) { a.top_value += (size_t)here * a.top; a.top_id += (size_t)here * a.top; }
    rows -= here;
    rest = 0;
  }
  return 0;
}
template <typename T, bool TOP>
static int launch_all(const LogprobArgs& a, int rows, int whole, int parts, cudaStream_t s) {
  const int rc = whole ? launch_rows<T, TOP>(a, 0, whole, 1, 0, s) : 0;
  return rc || whole == rows ? rc : launch_rows<T, TOP>(a, whole, rows - whole, parts, whole > 0, s);
}

extern "C" {

// logits: [rows, vocab], dtype 0 float, 1 bfloat16, rows `row_stride` entries apart; tokens [rows]; top 0 to 32, at most vocab;
// given, entropy [rows]; top_value, top_id [rows, top] (null with top 0).  The first `whole` rows have a block each,
// the others `parts` blocks (1, 2, 4 or 8); with alternatives a block takes at most 160 tiles of 16 KB.  A token of vocab or more sets bit
// 1 of *status (null: not told) and has no log probability.
int sb_token_logprobs(int dtype, const void* logits, int rows, int vocab, long long row_stride, const int* tokens, int top, float* given,
                      float* entropy, float* top_value, int* top_id, int whole, int parts, int* status, cudaStream_t s) {
  if (rows == 0) return 0;
  if (vocab < 1 || top < 0 || top > LP_MAX_TOP || top > vocab || row_stride < 0) return -2;
  if (parts != 1 && parts != 2 && parts != 4 && parts != LP_MAX_CLUSTER) return -2;
  if (whole < 0 || whole > rows) return -2;
  if (vocab > 0x7fff0000 || ((uintptr_t)logits & (dtype == 0 ? 3 : 1))) return -2;
  const LogprobArgs a{logits, row_stride, vocab, top, tokens, given, entropy, top_value, top_id, status};
  if (dtype == 0) return top ? launch_all<float, true>(a, rows, whole, parts, s) : launch_all<float, false>(a, rows, whole, parts, s);
  if (dtype == 1) return top ? launch_all<bf16, true>(a, rows, whole, parts, s) : launch_all<bf16, false>(a, rows, whole, parts, s);
  return -1;
}

}  // extern "C"
