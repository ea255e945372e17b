// Router, alone (ggo_moe_route) and with the balance loss, forward and backward.
//
// For every token t: the top_k experts of the fp32 logits l (ties to the lower index), their
// softmax weights, and the softmax P over ALL experts. Over the kept tokens (not masked, at least
// one logit above -inf; T' of them), with n_e the kept choices that fell on expert e:
//
//   f_e = n_e / (top_k T')     p_e = (1/T') sum_t P[t, e]     loss = E sum_e f_e p_e
//
// (1 for a balanced router). f is piecewise constant, so with g the loss's upstream gradient
//
//   d/dl[t, e] = g (E/T') P[t, e] (f_e - sum_e' P[t, e'] f_e')          (kept tokens)
//              + w_j (u_j - sum_j' w_j' u_j')   where e is token t's choice j, u = grad of w.
//
// Nothing here is accumulated by floating-point atomics: counts are integers, the sums over tokens
// go warp -> block -> a fixed-order reduction in 64 bits, so equal inputs give equal bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ggo.h"
#include "ggo_internal.h"

namespace ggo {
namespace {

constexpr int kTokens = 32;    // tokens per block: the granularity of the dispatch's offset table
constexpr int kMaxE = 1024;
constexpr int kMaxK = 16;
constexpr unsigned kAll = 0xffffffffu;

// Monotone float -> uint32 (larger float -> larger key). -0 counts as +0 and NaN as the largest, so
// that equal floats have equal keys; no float has key 0.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// A logit's key and its expert in one word, larger for larger logits and, among equal keys, for
// lower experts, so that a plain maximum chooses. The 16-bit types' keys are whole (upper half);
// fp32 keys lose their low 8 or 10 bits to the expert (IDX bits), which choose_top_k makes good.
template <typename TL>
struct KeyBits {
  static constexpr bool kWhole = true;
};
template <>
struct KeyBits<float> {
  static constexpr bool kWhole = false;
};

template <typename TL, int V>
__device__ __forceinline__ uint32_t packed_key(TL x, int e) {
  const float f = static_cast<float>(x);
  if constexpr (KeyBits<TL>::kWhole) {
    uint32_t b = *reinterpret_cast<const unsigned short*>(&x);
    if ((b & 0x7fffu) == 0) b = 0;  // -0 as +0
    const uint32_t key = f != f ? 0xffffu : ((b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u));
    return (key << 16) | (0xffffu - static_cast<uint32_t>(e));
  } else {
    constexpr uint32_t kIdx = V <= 8 ? 0xffu : 0x3ffu;
    return (order_key(f) & ~kIdx) | (kIdx - static_cast<uint32_t>(e));
  }
}
template <typename TL, int V>
__device__ __forceinline__ uint32_t index_mask() {
  return KeyBits<TL>::kWhole ? 0xffffu : (V <= 8 ? 0xffu : 0x3ffu);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Expert of a lane's i-th value: neighbouring experts on neighbouring lanes, or (VEC, E == 32 V) V
// neighbouring experts per lane, which are then loaded and stored 16 bytes at a time.
template <int V, bool VEC>
__device__ __forceinline__ int expert_of(int lane, int i) {
  return VEC ? lane * V + i : lane + 32 * i;
}

// A lane's values of one row of logits; values behind E are not defined.
template <typename TL, int V, bool VEC>
__device__ __forceinline__ void load_row(const TL* __restrict__ row, int E, int lane, TL (&x)[V]) {
  if constexpr (VEC) {
    constexpr int kBytes = V * static_cast<int>(sizeof(TL));
    const char* src = reinterpret_cast<const char*>(row) + lane * kBytes;
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(src)[i];
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(src);
    } else {
      *reinterpret_cast<uint32_t*>(x) = *reinterpret_cast<const uint32_t*>(src);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane + 32 * i < E) x[i] = row[lane + 32 * i];
  }
}

// The K largest logits of a row, lane j getting expert and logit of the j-th, by K maxima over the
// warp of whole (key, expert) pairs: exact for every input, and slow.
template <typename TL, int V>
__device__ __noinline__ int choose_exactly(const TL* __restrict__ row, int E, int K, int lane) {
  uint32_t key[V];
#pragma unroll
  for (int i = 0; i < V; ++i)
    key[i] = lane + 32 * i < E ? order_key(static_cast<float>(row[lane + 32 * i])) : 0u;
  int id = 0;
  for (int j = 0; j < K; ++j) {
    uint32_t m = key[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = max(m, key[i]);
    const uint32_t best = __reduce_max_sync(kAll, m);
    int e_min = kMaxE;
#pragma unroll
    for (int i = V - 1; i >= 0; --i)
      if (key[i] == best) e_min = lane + 32 * i;
    const int chosen = __reduce_min_sync(kAll, e_min);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane + 32 * i == chosen) key[i] = 0u;
    if (lane == j) id = chosen;
  }
  return id;
}

// Sorts a lane's V words in descending order (Batcher's odd-even merge sort; V a power of two).
template <int V>
__device__ __forceinline__ void sort_descending(uint32_t (&k)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < V; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t hi = max(k[i + j], k[i + j + q]), lo = min(k[i + j], k[i + j + q]);
            k[i + j] = hi;
            k[i + j + q] = lo;
          }
}

// The expert (lane j: the j-th choice) of the K largest of the warp's packed keys. With V <= 8 every
// lane sorts its keys once and the warp takes K times the largest head; longer lists are searched
// each time. fp32: a lost key bit matters only where two neighbours of the order, up to the first
// one not chosen, share the kept bits; then the row is chosen again with whole keys.
template <typename TL, int V>
__device__ __forceinline__ int choose_top_k(uint32_t (&k)[V], const TL* __restrict__ row, int E,
                                            int K, int lane) {
  constexpr bool kSorted = V <= 8;
  const uint32_t idx = index_mask<TL, V>();
  if constexpr (kSorted) sort_descending<V>(k);
  uint32_t mine = 0;
  const int rounds = KeyBits<TL>::kWhole ? K : K + 1;
  for (int j = 0; j < rounds; ++j) {
    uint32_t m = k[0];
    if constexpr (!kSorted) {
#pragma unroll
      for (int i = 1; i < V; ++i) m = max(m, k[i]);
    }
    const uint32_t best = __reduce_max_sync(kAll, m);
    if constexpr (kSorted) {
      const bool pop = m == best;
#pragma unroll
      for (int i = 0; i + 1 < V; ++i) k[i] = pop ? k[i + 1] : k[i];
      k[V - 1] = pop ? 0u : k[V - 1];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) k[i] = k[i] == best ? 0u : k[i];
    }
    if (lane == j) mine = best;
  }
  int id = static_cast<int>(idx - (mine & idx));
  if constexpr (!KeyBits<TL>::kWhole) {
    const uint32_t next = __shfl_down_sync(kAll, mine, 1);
    const bool unsure = lane < K && ((mine ^ next) & ~idx) == 0;
    if (__any_sync(kAll, unsure)) id = choose_exactly<TL, V>(row, E, K, lane);
  }
  return id;
}

// What one block makes of its tokens, a warp each at a time (NW warps; tokens t0 + warp, + NW, ...):
// ids, weights and row_stat[t] = (max logit, 1 / sum exp(l - max)), the second 0 for tokens that are
// not kept; in shared memory hist[e], the block's choices of expert e, all in the low and kept in the
// high 16 bits, and wsum[warp][e], the warps' sums of P over kept tokens. Ends with a barrier.
// Without LOSS: ids, weights and hist only.
template <typename TL, int V, bool VEC, int NW, bool LOSS>
__device__ __forceinline__ void route_block(const TL* __restrict__ logits,
                                            const uint8_t* __restrict__ mask, int T, int E, int K,
                                            int32_t* __restrict__ ids, float* __restrict__ weights,
                                            float2* __restrict__ row_stat, int t0, uint32_t* hist,
                                            float* wsum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < E; e += 32 * NW) hist[e] = 0;
  __syncthreads();
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  const int ntok = min(T - t0, kTokens);  // (t0 + kTokens may pass 32 bits; t0 < T)
  for (int tl = warp; tl < ntok; tl += NW) {
    const int t = t0 + tl;
    const TL* row = logits + static_cast<size_t>(t) * E;
    alignas(16) TL x[V];
    load_row<TL, V, VEC>(row, E, lane, x);
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = expert_of<V, VEC>(lane, i);
      key[i] = (VEC || e < E) ? packed_key<TL, V>(x[i], e) : 0u;
    }
    const int id = choose_top_k<TL, V>(key, row, E, K, lane);
    const float val = lane < K ? static_cast<float>(row[id]) : 0.f;
    const float top = __shfl_sync(kAll, val, 0);
    const bool live = top != -INFINITY;
    const bool kept = live && (mask == nullptr || mask[t] != 0);
    // softmax over the choices, summed in choice order
    const float ex = (lane < K && live) ? expf(val - top) : 0.f;
    float s = 0.f;
    for (int j = 0; j < K; ++j) s += __shfl_sync(kAll, ex, j);
    const float inv_k = live ? 1.0f / s : 0.f;
    if (lane < K) {
      ids[static_cast<size_t>(t) * K + lane] = id;
      weights[static_cast<size_t>(t) * K + lane] = ex * inv_k;
      atomicAdd(&hist[id], kept ? 0x10001u : 1u);
    }
    // softmax over all experts
    float inv = 0.f;
    if (LOSS && kept) {
      float p[V];
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        p[i] = (VEC || lane + 32 * i < E) ? expf(static_cast<float>(x[i]) - top) : 0.f;
        z += p[i];
      }
      inv = 1.0f / warp_sum(z);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(p[i], inv, acc[i]);
    }
    if (LOSS && lane == 0) row_stat[t] = make_float2(live ? top : 0.f, inv);
  }
  if constexpr (LOSS) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = expert_of<V, VEC>(lane, i);
      if (VEC || e < E) wsum[warp * E + e] = acc[i];
    }
  }
  __syncthreads();
}

// The first of two launches. grid = ceil(T / kTokens), NW warps: 8, or 32 (a token each) when the blocks
// would not fill the GPU. table[b][e] and psum[b][e] receive block b's hist and its sum of P. 32768 x 256
// in bf16: 25 us, of which reading takes 3 and issuing the 580 instructions a token 16 (70 % of the issue
// slots are used, 48 % of the warps resident); the rest is the wait of each of the k maxima for the one
// before.
template <typename TL, int V, bool VEC, int NW, bool LOSS>
__global__ void __launch_bounds__(32 * NW)
    router_kernel(const TL* __restrict__ logits, const uint8_t* __restrict__ mask, int T, int E,
                  int K, int32_t* __restrict__ ids, float* __restrict__ weights,
                  float2* __restrict__ row_stat, uint32_t* __restrict__ table,
                  float* __restrict__ psum) {
  extern __shared__ uint32_t sm[];
  uint32_t* hist = sm;                                    // [E]
  float* wsum = reinterpret_cast<float*>(sm + E);         // [NW][E]
  route_block<TL, V, VEC, NW, LOSS>(logits, mask, T, E, K, ids, weights, row_stat,
                                    blockIdx.x * kTokens, hist, wsum);
  for (int e = threadIdx.x; e < E; e += 32 * NW) {
    if constexpr (LOSS) {
      float p = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) p += wsum[w * E + e];
      psum[static_cast<size_t>(blockIdx.x) * E + e] = p;
    }
    table[static_cast<size_t>(blockIdx.x) * E + e] = hist[e];
  }
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

// Over the experts, thread e of 1024 giving expert e's choices, kept choices and sum of P (threads
// behind E zeros): the exclusive sum of the choices, and of all the kept choices and n_e sum P. Within
// warps, then over the warps' sums: the order is fixed. Contains a barrier.
struct ExpertScan {
  int start;
  long long choices;  // top_k T'
  double sum_np;      // sum_e n_e sum_t P
};

__device__ __forceinline__ ExpertScan scan_experts(int mine, int mine_kept, double p, int E) {
  __shared__ int warp_tot[32], warp_kept[32];
  __shared__ double warp_term[32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  double term = static_cast<double>(mine_kept) * p;
  int scan = mine, ksum = mine_kept;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kAll, scan, o);
    if (lane >= o) scan += v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ksum += __shfl_xor_sync(kAll, ksum, o);
    term += __shfl_xor_sync(kAll, term, o);
  }
  if (lane == 31) {
    warp_tot[wid] = scan;
    warp_kept[wid] = ksum;
    warp_term[wid] = term;
  }
  __syncthreads();
  ExpertScan r{scan - mine, 0, 0.0};
  for (int w = 0; w < (E + 31) / 32; ++w) {
    if (w < wid) r.start += warp_tot[w];
    r.choices += warp_kept[w];
    r.sum_np += warp_term[w];
  }
  return r;
}

// loss = E sum_e (n_e / choices) (sum_t P / T'), T' = choices / K. The gradient takes f only through
// f_e - sum P f, which a constant added to f does not change: coef_e = E (f_e - 1/E) / T', so that a
// nearly balanced router's small gradient is not the difference of two large numbers. Without LOSS: the
// experts' counts only.
template <bool LOSS>
__device__ __forceinline__ void write_totals(const ExpertScan& sc, int mine, int mine_kept, int E,
                                             int K, int64_t* __restrict__ tpe,
                                             int64_t* __restrict__ kept_counts,
                                             float* __restrict__ loss, float* __restrict__ coef) {
  const int tid = threadIdx.x;
  if (tid < E) tpe[tid] = mine;
  if (!LOSS) return;
  const double n = static_cast<double>(sc.choices);
  const double scale = sc.choices > 0 ? static_cast<double>(E) * K / (n * n) : 0.0;
  if (tid < E) {
    kept_counts[tid] = mine_kept;
    coef[tid] = static_cast<float>(scale * (mine_kept - n / E));
  }
  if (tid == 0) *loss = static_cast<float>(scale * sc.sum_np);
}

// The whole forward in one launch, for up to 8 x 32 tokens and 256 experts: one cluster, a block of 32
// warps per 32 tokens, a token each. The blocks hand one another their counts and sums through
// distributed shared memory and each writes its row of the offset table. 256 x 256 in fp32: 8.7 us; two
// launches for one token more, 11.6.
constexpr int kSmallBlocks = 8;
template <typename TL, int V, bool VEC, bool LOSS>
__global__ void __launch_bounds__(1024)
    router_small_kernel(const TL* __restrict__ logits, const uint8_t* __restrict__ mask, int T,
                        int E, int K, int32_t* __restrict__ ids, float* __restrict__ weights,
                        float2* __restrict__ row_stat, int* __restrict__ table,
                        int64_t* __restrict__ tpe, int64_t* __restrict__ kept_counts,
                        float* __restrict__ loss, float* __restrict__ coef) {
  extern __shared__ uint32_t sm[];
  uint32_t* hist = sm;                             // [E]
  float* wsum = reinterpret_cast<float*>(sm + E);  // [32][E], then [2][kSmallBlocks][E]
  const int tid = threadIdx.x;
  unsigned rank, nblocks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(nblocks));
  route_block<TL, V, VEC, 32, LOSS>(logits, mask, T, E, K, ids, weights, row_stat, rank * kTokens,
                                    hist, wsum);
  float p = 0.f;
  if (LOSS && tid < E) {
#pragma unroll
    for (int w = 0; w < 32; ++w) p += wsum[w * E + tid];
  }
  cluster_barrier();  // every block has read its wsum: the room is now the mailboxes
  if (tid < E) {
    const uint32_t box = static_cast<uint32_t>(
        __cvta_generic_to_shared(wsum + rank * static_cast<unsigned>(E) + tid));
    for (unsigned r = 0; r < nblocks; ++r) {
      uint32_t to;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(box), "r"(r));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(hist[tid]) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + kSmallBlocks * E * 4), "f"(p)
                   : "memory");
    }
  }
  cluster_barrier();
  const uint32_t* counts = reinterpret_cast<const uint32_t*>(wsum);
  const float* sums = wsum + kSmallBlocks * E;
  int all = 0, kept = 0, before = 0;
  double ps = 0.0;
  if (tid < E) {
    for (unsigned r = 0; r < nblocks; ++r) {
      const uint32_t v = counts[r * E + tid];
      if (r < rank) before += v & 0xffffu;
      all += v & 0xffffu;
      kept += v >> 16;
      ps += sums[r * E + tid];
    }
  }
  const ExpertScan sc = scan_experts(all, kept, ps, E);
  if (tid < E) {
    table[rank * E + tid] = sc.start + before;
    if (rank == 0) table[nblocks * E + tid] = sc.start;
  }
  if (rank == 0) write_totals<LOSS>(sc, all, kept, E, K, tpe, kept_counts, loss, coef);
}

// One cluster of up to 8 CTAs x 1024 threads; CTA r owns experts [r * CE, (r+1) * CE). Thread
// (q, c) = (tid / CP, tid % CP), q < R, walks rows [q * per, (q+1) * per) of expert column c, so that
// a warp reads 32 neighbouring experts. R is at most 32: one thread per expert adds the ranges up. Totals are exchanged through distributed shared memory.
// 32768 x 256: 15 us, the eight SMs' share of L2 bandwidth over two passes; 256 x 256: 5 us.
// Turns table into the dispatch's absolute start rows (in place, expert starts right behind it) and
// writes the counts and, with LOSS, the loss and coef[e] = E (f_e - 1/E) / T' for the backward.
template <bool LOSS>
__global__ void __launch_bounds__(1024)
    router_finish_kernel(uint32_t* __restrict__ table, const float* __restrict__ psum, int nblocks,
                         int E, int K, int CE, int CP, int64_t* __restrict__ tpe,
                         int64_t* __restrict__ kept_counts, float* __restrict__ loss,
                         float* __restrict__ coef) {
  __shared__ int part_all[1024];     // [R][CP] range sums, then exclusive offsets of the ranges
  __shared__ int part_kept[1024];
  __shared__ double part_p[1024];
  __shared__ int tot[kMaxE];         // every expert's totals (gathered from the whole cluster)
  __shared__ int tot_kept[kMaxE];
  __shared__ double tot_p[kMaxE];
  __shared__ int start[kMaxE];
  unsigned rank, ncta;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ncta));
  const int tid = threadIdx.x;
  const int R = min(1024 / CP, 32);
  const int c = tid % CP, q = tid / CP;
  const int e = static_cast<int>(rank) * CE + c;
  const bool active = c < CE && e < E;
  const int per = (nblocks + R - 1) / R;
  const int b0 = min(nblocks, q * per), b1 = min(nblocks, b0 + per);
  int all = 0, kept = 0;
  double p = 0.0;
  if (active) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
      const uint32_t v = table[static_cast<size_t>(b) * E + e];
      all += v & 0xffffu;
      kept += v >> 16;
      if (LOSS) p += psum[static_cast<size_t>(b) * E + e];
    }
  }
  part_all[tid] = all;
  part_kept[tid] = kept;
  part_p[tid] = p;
  __syncthreads();
  cluster_barrier();  // every CTA of the cluster runs before its shared memory is written
  // totals of expert e (q == 0: this thread's own), scanned over its ranges, into every CTA
  if (tid < CP && active) {
    int run = 0, ksum = 0;
    double ps = 0.0;
    for (int j = 0; j < R; ++j) {
      const int v = part_all[j * CP + c];
      part_all[j * CP + c] = run;
      run += v;
      ksum += part_kept[j * CP + c];
      ps += part_p[j * CP + c];
    }
    for (unsigned r = 0; r < ncta; ++r) {
      uint32_t a, b, d;
      const uint32_t la = static_cast<uint32_t>(__cvta_generic_to_shared(&tot[e]));
      const uint32_t lb = static_cast<uint32_t>(__cvta_generic_to_shared(&tot_kept[e]));
      const uint32_t ld = static_cast<uint32_t>(__cvta_generic_to_shared(&tot_p[e]));
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(la), "r"(r));
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(lb), "r"(r));
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(ld), "r"(r));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(run) : "memory");
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(b), "r"(ksum) : "memory");
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(d), "d"(ps) : "memory");
    }
  }
  cluster_barrier();
  const int mine = tid < E ? tot[tid] : 0;
  const int mine_kept = tid < E ? tot_kept[tid] : 0;
  const ExpertScan sc = scan_experts(mine, mine_kept, tid < E ? tot_p[tid] : 0.0, E);
  start[tid] = sc.start;
  __syncthreads();
  if (active) {
    const int first = start[e];
    if (q == 0) reinterpret_cast<int*>(table)[static_cast<size_t>(nblocks) * E + e] = first;
    int run = first + part_all[tid];
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
      const size_t i = static_cast<size_t>(b) * E + e;
      const int v = table[i] & 0xffffu;
      table[i] = static_cast<uint32_t>(run);
      run += v;
    }
  }
  if (rank == 0) write_totals<LOSS>(sc, mine, mine_kept, E, K, tpe, kept_counts, loss, coef);
}

// One warp per token, persistent over tokens so that a lane's coefficients stay in registers. Every
// warp owns E floats of shared memory in which the k choices' gradients are laid out by expert.
constexpr int kBwdWarps = 8;
// Blocks that run at once on an SM (by registers). The grid is one wave of them: 32768 x 256 in bf16
// 15.8 us, 18.1 us with a grid of 1.3 waves. The kernel issues 300 instructions a token, a third of
// them in expf, in 8 of its microseconds; its bytes would take 5. The rest is waiting: two warp sums
// in a row for every token.
constexpr int bwd_blocks(int v) { return v <= 8 ? 6 : (v == 16 ? 3 : 2); }

template <typename TL, int V, bool VEC>
__global__ void __launch_bounds__(32 * kBwdWarps, bwd_blocks(V))
    router_backward_kernel(const TL* __restrict__ logits, const float2* __restrict__ row_stat,
                           const int32_t* __restrict__ ids, const float* __restrict__ weights,
                           const float* __restrict__ coef, const float* __restrict__ grad_w,
                           const float* __restrict__ grad_loss, int T, int E, int K,
                           TL* __restrict__ out) {
  extern __shared__ uint32_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* add = reinterpret_cast<float*>(sm) + warp * E;
  for (int e = lane; e < E; e += 32) add[e] = 0.f;
  const float gl = grad_loss ? *grad_loss : 0.f;
  float cf[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = expert_of<V, VEC>(lane, i);
    cf[i] = (VEC || e < E) ? gl * coef[e] : 0.f;
  }
  __syncwarp();
  // unsigned: the step past the last token may lie behind 2^31
  for (unsigned t = blockIdx.x * kBwdWarps + warp; t < static_cast<unsigned>(T);
       t += gridDim.x * kBwdWarps) {
    const float2 st = row_stat[t];
    alignas(16) TL x[V];
    load_row<TL, V, VEC>(logits + static_cast<size_t>(t) * E, E, lane, x);
    int id = 0;
    if (grad_w) {
      float w = 0.f, u = 0.f;
      if (lane < K) {
        id = ids[static_cast<size_t>(t) * K + lane];
        w = weights[static_cast<size_t>(t) * K + lane];
        u = grad_w[static_cast<size_t>(t) * K + lane];
      }
      const float mean = warp_sum(w * u);
      if (lane < K) add[id] = w * (u - mean);
      __syncwarp();
    }
    float p[V];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool some = (VEC || lane + 32 * i < E) && st.y != 0.f;
      p[i] = some ? expf(static_cast<float>(x[i]) - st.x) * st.y : 0.f;
      dot = fmaf(p[i], cf[i], dot);
    }
    dot = warp_sum(dot);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = expert_of<V, VEC>(lane, i);
      if (VEC || e < E) x[i] = static_cast<TL>(fmaf(p[i], cf[i] - dot, add[e]));
    }
    TL* dst = out + static_cast<size_t>(t) * E;
    if constexpr (VEC) {
      constexpr int kBytes = V * static_cast<int>(sizeof(TL));
      char* d = reinterpret_cast<char*>(dst) + lane * kBytes;
      if constexpr (kBytes >= 16) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i)
          reinterpret_cast<uint4*>(d)[i] = reinterpret_cast<const uint4*>(x)[i];
      } else if constexpr (kBytes == 8) {
        *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(x);
      } else {
        *reinterpret_cast<uint32_t*>(d) = *reinterpret_cast<const uint32_t*>(x);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (lane + 32 * i < E) dst[lane + 32 * i] = x[i];
    }
    if (grad_w) {
      __syncwarp();
      if (lane < K) add[id] = 0.f;
      __syncwarp();
    }
  }
}

int blocks_for(int64_t T) { return static_cast<int>((T + kTokens - 1) / kTokens); }

// Sixteen-byte access to rows needs rows and base on 16-byte boundaries: E == 32 V with at least four
// bytes per lane, on an aligned tensor.
template <typename TL, int V>
bool vec_rows(const void* a, const void* b, int E) {
  return E == 32 * V && V * sizeof(TL) >= 4 &&
         ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) == 0;
}

template <typename TL, int V, bool VEC, int NW, bool LOSS>
int launch_router_as(const void* logits, const uint8_t* mask, int T, int E, int K, int32_t* ids,
                     float* w, float2* stat, uint32_t* table, float* psum, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(E) * (1 + NW) * 4;  // at most 36 KB
  router_kernel<TL, V, VEC, NW, LOSS><<<blocks_for(T), 32 * NW, smem, stream>>>(
      static_cast<const TL*>(logits), mask, T, E, K, ids, w, stat, table, psum);
  return check_launch();
}

// A warp per token while the blocks find free SMs; beyond that eight warps of four tokens each.
// 256 tokens x 256 experts, fp32: 5.6 us against 16.5 us with eight warps of four tokens.
constexpr int kWideBlocks = 148;

template <typename TL, int V, bool VEC, bool LOSS>
int launch_router_vec(const void* logits, const uint8_t* mask, int T, int E, int K, int32_t* ids,
                      float* w, float2* stat, uint32_t* table, float* psum, cudaStream_t stream) {
  if constexpr (V <= 8)
    if (blocks_for(T) <= kWideBlocks)
      return launch_router_as<TL, V, VEC, 32, LOSS>(logits, mask, T, E, K, ids, w, stat, table,
                                                    psum, stream);
  return launch_router_as<TL, V, VEC, 8, LOSS>(logits, mask, T, E, K, ids, w, stat, table, psum,
                                               stream);
}

template <typename TL, int V, bool LOSS = true>
int launch_router(const void* logits, const uint8_t* mask, int T, int E, int K, int32_t* ids,
                  float* w, float2* stat, uint32_t* table, float* psum, cudaStream_t stream) {
  if constexpr (V * sizeof(TL) >= 4)
    if (vec_rows<TL, V>(logits, nullptr, E))
      return launch_router_vec<TL, V, true, LOSS>(logits, mask, T, E, K, ids, w, stat, table, psum,
                                                  stream);
  return launch_router_vec<TL, V, false, LOSS>(logits, mask, T, E, K, ids, w, stat, table, psum,
                                               stream);
}

template <typename TL, int V, bool VEC, bool LOSS>
int launch_small_as(const void* logits, const uint8_t* mask, int T, int E, int K, int32_t* ids,
                    float* w, float2* stat, int* table, int64_t* tpe, int64_t* kept, float* loss,
                    float* coef, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks_for(T), 1, 1);
  cfg.blockDim = dim3(1024, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(E) * 33 * 4;  // at most 33 KB
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks_for(T);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, router_small_kernel<TL, V, VEC, LOSS>,
                                         static_cast<const TL*>(logits), mask, T, E, K, ids, w,
                                         stat, table, tpe, kept, loss, coef))
    return cuda_fail(static_cast<int>(e));
  return check_launch();
}

template <typename TL, int V, bool LOSS = true>
int launch_small(const void* logits, const uint8_t* mask, int T, int E, int K, int32_t* ids,
                 float* w, float2* stat, int* table, int64_t* tpe, int64_t* kept, float* loss,
                 float* coef, cudaStream_t stream) {
  if constexpr (V > 8) {
    return GGO_ERR_SHAPE;
  } else {
    if constexpr (V * sizeof(TL) >= 4)
      if (vec_rows<TL, V>(logits, nullptr, E))
        return launch_small_as<TL, V, true, LOSS>(logits, mask, T, E, K, ids, w, stat, table, tpe,
                                                  kept, loss, coef, stream);
    return launch_small_as<TL, V, false, LOSS>(logits, mask, T, E, K, ids, w, stat, table, tpe,
                                               kept, loss, coef, stream);
  }
}

template <typename TL, int V, bool VEC>
int launch_backward_as(const void* logits, const float2* stat, const int32_t* ids, const float* w,
                       const float* coef, const float* gw, const float* gl, int T, int E, int K,
                       void* out, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(E) * kBwdWarps * 4;
  const int want = (T - 1) / kBwdWarps + 1;  // T > 0; T + 7 may pass 32 bits
  const int wave = 148 * bwd_blocks(V);
  const int grid = want < wave ? want : wave;
  router_backward_kernel<TL, V, VEC><<<grid, 32 * kBwdWarps, smem, stream>>>(
      static_cast<const TL*>(logits), stat, ids, w, coef, gw, gl, T, E, K, static_cast<TL*>(out));
  return check_launch();
}

template <typename TL, int V>
int launch_backward(const void* logits, const float2* stat, const int32_t* ids, const float* w,
                    const float* coef, const float* gw, const float* gl, int T, int E, int K,
                    void* out, cudaStream_t stream) {
  if constexpr (V * sizeof(TL) >= 4)
    if (vec_rows<TL, V>(logits, out, E))
      return launch_backward_as<TL, V, true>(logits, stat, ids, w, coef, gw, gl, T, E, K, out,
                                             stream);
  return launch_backward_as<TL, V, false>(logits, stat, ids, w, coef, gw, gl, T, E, K, out,
                                          stream);
}

// Calls f<TL, V>() with TL by dtype and V the smallest power of two that holds ceil(E / 32).
#define GGO_ROUTER_CALL_V(TL, FN, ...)                          \
  (E <= 32    ? FN<TL, 1>(__VA_ARGS__)                          \
   : E <= 64  ? FN<TL, 2>(__VA_ARGS__)                          \
   : E <= 128 ? FN<TL, 4>(__VA_ARGS__)                          \
   : E <= 256 ? FN<TL, 8>(__VA_ARGS__)                          \
   : E <= 512 ? FN<TL, 16>(__VA_ARGS__)                         \
              : FN<TL, 32>(__VA_ARGS__))
#define GGO_ROUTER_CALL(FN, ...)                                             \
  (dtype == GGO_DTYPE_FP32   ? GGO_ROUTER_CALL_V(float, FN, __VA_ARGS__)     \
   : dtype == GGO_DTYPE_BF16 ? GGO_ROUTER_CALL_V(__nv_bfloat16, FN, __VA_ARGS__) \
                             : GGO_ROUTER_CALL_V(__half, FN, __VA_ARGS__))

bool router_args_ok(int64_t num_tokens, int num_experts, int top_k) {
  return num_tokens >= 0 && num_experts > 0 && num_experts <= kMaxE && top_k > 0 &&
         top_k <= kMaxK && top_k <= num_experts;
}

bool router_dtype_ok(int dtype) {
  return dtype == GGO_DTYPE_FP32 || dtype == GGO_DTYPE_BF16 || dtype == GGO_DTYPE_FP16;
}

// Routing without the loss, of fp32 logits.
template <typename TL, int V>
int launch_route(const void* logits, int T, int E, int K, int32_t* ids, float* w, uint32_t* table,
                 cudaStream_t stream) {
  return launch_router<TL, V, false>(logits, nullptr, T, E, K, ids, w, nullptr, table, nullptr,
                                     stream);
}

template <typename TL, int V>
int launch_route_small(const void* logits, int T, int E, int K, int32_t* ids, float* w,
                       int* table, int64_t* tpe, cudaStream_t stream) {
  return launch_small<TL, V, false>(logits, nullptr, T, E, K, ids, w, nullptr, table, tpe, nullptr,
                                    nullptr, nullptr, stream);
}

// Whether one launch does the whole routing.
bool small_routing(int nb, int E) { return nb > 0 && nb <= kSmallBlocks && E <= 256; }

template <bool LOSS>
int launch_finish(uint32_t* table, const float* psum, int nb, int E, int K, int64_t* tpe,
                  int64_t* kept, float* loss, float* coef, cudaStream_t stream) {
  // experts per CTA: 32 (a coalesced row piece), or E / 8 beyond 256 experts
  int ncta = 1;
  while (ncta < 8 && ncta * 32 < E) ncta *= 2;
  const int CE = (E + ncta - 1) / ncta;
  int CP = 1;
  while (CP < CE) CP *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ncta, 1, 1);
  cfg.blockDim = dim3(1024, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ncta;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, router_finish_kernel<LOSS>, table, psum, nb, E, K,
                                         CE, CP, tpe, kept, loss, coef))
    return cuda_fail(static_cast<int>(e));
  return check_launch();
}

}  // namespace
}  // namespace ggo

extern "C" {

size_t ggo_moe_router_scratch_bytes(int64_t num_tokens, int num_experts) {
  if (num_tokens < 0 || num_experts <= 0) return 16;
  // the dispatch's table and expert starts (as ggo_moe_route_scratch_bytes), then the sums of P
  return (2 * static_cast<size_t>(ggo::blocks_for(num_tokens)) + 1) * num_experts * 4;
}

int ggo_moe_router(const void* logits_dev, int dtype, int64_t num_tokens, int num_experts,
                   int top_k, const uint8_t* token_mask_dev, int32_t* topk_ids_dev,
                   float* topk_weights_dev, int64_t* tokens_per_expert_dev,
                   int64_t* balance_counts_dev, float* balance_loss_dev, float* row_stat_dev,
                   float* coef_dev, void* scratch_dev, cudaStream_t stream) {
  if (!ggo::router_args_ok(num_tokens, num_experts, top_k)) return GGO_ERR_INVALID_ARG;
  if (!tokens_per_expert_dev || !balance_counts_dev || !balance_loss_dev || !coef_dev ||
      !scratch_dev)
    return GGO_ERR_INVALID_ARG;
  if (num_tokens > 0 && (!logits_dev || !topk_ids_dev || !topk_weights_dev || !row_stat_dev))
    return GGO_ERR_INVALID_ARG;
  if (!ggo::router_dtype_ok(dtype)) return GGO_ERR_DTYPE;
  if (num_tokens * top_k > INT32_MAX) return GGO_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(row_stat_dev) & 7u) ||
      (reinterpret_cast<uintptr_t>(scratch_dev) & 3u))
    return GGO_ERR_ALIGNMENT;
  const int T = static_cast<int>(num_tokens), E = num_experts;
  const int nb = ggo::blocks_for(num_tokens);
  uint32_t* table = static_cast<uint32_t*>(scratch_dev);
  float* psum = reinterpret_cast<float*>(table + (static_cast<size_t>(nb) + 1) * E);
  float2* stat = reinterpret_cast<float2*>(row_stat_dev);
  if (ggo::small_routing(nb, E))
    return GGO_ROUTER_CALL(ggo::launch_small, logits_dev, token_mask_dev, T, E, top_k,
                           topk_ids_dev, topk_weights_dev, stat, reinterpret_cast<int*>(table),
                           tokens_per_expert_dev, balance_counts_dev, balance_loss_dev, coef_dev,
                           stream);
  if (nb > 0) {
    const int st = GGO_ROUTER_CALL(ggo::launch_router, logits_dev, token_mask_dev, T, E, top_k,
                                   topk_ids_dev, topk_weights_dev, stat, table, psum, stream);
    if (st) return st;
  }
  return ggo::launch_finish<true>(table, psum, nb, E, top_k, tokens_per_expert_dev,
                                  balance_counts_dev, balance_loss_dev, coef_dev, stream);
}

int ggo_moe_route(const float* logits_dev, int64_t num_tokens, int num_experts, int top_k,
                  int32_t* topk_ids_dev, float* topk_weights_dev,
                  int64_t* tokens_per_expert_dev, void* scratch_dev, cudaStream_t stream) {
  if (!tokens_per_expert_dev || !scratch_dev ||
      (num_tokens != 0 && (!logits_dev || !topk_ids_dev || !topk_weights_dev)))
    return GGO_ERR_INVALID_ARG;
  if (!ggo::router_args_ok(num_tokens, num_experts, top_k)) return GGO_ERR_INVALID_ARG;
  if (num_tokens * top_k > INT32_MAX) return GGO_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(scratch_dev) & 3u) return GGO_ERR_ALIGNMENT;
  const int T = static_cast<int>(num_tokens), E = num_experts;
  const int nb = ggo::blocks_for(num_tokens);
  uint32_t* table = static_cast<uint32_t*>(scratch_dev);
  if (ggo::small_routing(nb, E))
    return GGO_ROUTER_CALL_V(float, ggo::launch_route_small, logits_dev, T, E, top_k, topk_ids_dev,
                             topk_weights_dev, reinterpret_cast<int*>(table),
                             tokens_per_expert_dev, stream);
  if (nb > 0) {
    const int st = GGO_ROUTER_CALL_V(float, ggo::launch_route, logits_dev, T, E, top_k,
                                     topk_ids_dev, topk_weights_dev, table, stream);
    if (st) return st;
  }
  return ggo::launch_finish<false>(table, nullptr, nb, E, top_k, tokens_per_expert_dev, nullptr,
                                   nullptr, nullptr, stream);
}

int ggo_moe_router_backward(const void* logits_dev, int dtype, int64_t num_tokens, int num_experts,
                            int top_k, const int32_t* topk_ids_dev, const float* topk_weights_dev,
                            const float* row_stat_dev, const float* coef_dev,
                            const float* grad_weights_dev, const float* grad_loss_dev,
                            void* grad_logits_dev, cudaStream_t stream) {
  if (!ggo::router_args_ok(num_tokens, num_experts, top_k)) return GGO_ERR_INVALID_ARG;
  if (!ggo::router_dtype_ok(dtype)) return GGO_ERR_DTYPE;
  if (num_tokens * top_k > INT32_MAX) return GGO_ERR_SHAPE;
  if (num_tokens == 0) return GGO_OK;
  if (!logits_dev || !topk_ids_dev || !topk_weights_dev || !row_stat_dev || !coef_dev ||
      !grad_logits_dev)
    return GGO_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(row_stat_dev) & 7u) return GGO_ERR_ALIGNMENT;
  const int T = static_cast<int>(num_tokens), E = num_experts;
  return GGO_ROUTER_CALL(ggo::launch_backward, logits_dev,
                         reinterpret_cast<const float2*>(row_stat_dev), topk_ids_dev,
                         topk_weights_dev, coef_dev, grad_weights_dev, grad_loss_dev, T, E, top_k,
                         grad_logits_dev, stream);
}

}  // extern "C"
