// The router of a mixture of experts: top-k choice, weights, the order of rows by expert, the load-balancing term, and the
// gradient of weights and term.
//
// Per token, logits l over E experts, k of them chosen in falling order (ties to the lowest index):
//   w_j = exp(l_j) / sum over the chosen of exp(l_i),  p = softmax(l),  aux = E sum_e share_e mean_t p[t, e]
//   dl[t, e_j] += w_j (dw_j - sum_i w_i dw_i),  dl[t, e] += daux E / T p[t, e] (share_e - sum_i share_i p[t, i])
// with share_e = choices made for e / (T k).
//
// A token belongs to a group of LANES threads (the power of two that holds E, 32 at most, VALS logits each), which finds one choice
// per round with two warp reductions: the largest key (floats as ordered integers), then the lowest index that has it (bf16 keys carry
// their index: one reduction).  Up to four logits of a lane are sorted once, so that a round looks at its first only.  Rows are
// numbered by a counting sort that keeps the order of the choices inside an expert: every CTA counts the choices of a run of
// consecutive tokens; the second kernel adds up the counts before its own run and ranks its choices.  No float atomics: the sums of p
// are added in a fixed order.  Few tokens take one launch of one CTA, which keeps the choices in shared memory.
//
// Bound by latency (chains of warp reductions, counts that wait for counts), not by its few bytes: 8192 tokens x 8 experts, 2 choices 5.5 us and
// 5.6 for the rows; 16389 x 128, 8 choices, 5 MB, 13 and 9; one token 5.7; the gradient 6 and 10.8.
#include "common.cuh"
#include "moe_api.h"

namespace tb {

namespace {

constexpr int kThreads = 1024;      // of the forward kernels: one CTA per SM, and its latencies have 32 warps to hide behind
constexpr int kBwdThreads = 256;
constexpr int kWarps = kThreads / 32;
static_assert(kWarps == 32, "a lane per warp");
constexpr int kMaxChunks = 148;

__device__ __forceinline__ uint32_t to_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);      // -0 and 0 tie
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_key(uint32_t k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }
constexpr uint32_t kKeyMinusInf = 0x007fffffu;      // to_key(-inf); 0: taken, or past the last expert

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

template <int LANES>
__device__ __forceinline__ uint32_t group_mask(int lane) {
  return LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
}
template <int LANES>
__device__ __forceinline__ float group_sum(float v, uint32_t mask) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o, LANES);
  return v;
}

struct RouteArgs {
  int64_t ld;
  int T, E, k, capacity;
  int chunk;               // tokens of a CTA
  float* weights;
  int* experts;
  int* slots;
  int* offsets;
  int* rows;
  int* counts;
  float* aux;
  int* hist;               // [chunks][E]
  float* psum;             // [chunks][E]
};

// Numbers the choices of CTA `c` of `chunks`.  codes: the expert of each of its choices (-1: not made), from its first on.
__device__ void plan_rows(const RouteArgs& a, const int* codes, const int* all_hist, const float* all_psum, int c, int chunks, int* sm) {
  const int E = a.E, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* total = sm;                 // [E]
  int* before = sm + E;            // [E] in earlier CTAs
  int* first = sm + 2 * E;         // [E + 1] first row of each expert
  const int S = E | 1;             // an odd stride: the counts of an expert lie in different banks
  int* cnt = sm + 3 * E + 1;       // [kWarps][S]
  float* aux_part = reinterpret_cast<float*>(cnt + kWarps * S);      // [kWarps]
  for (int i = tid; i < 2 * E; i += kThreads) sm[i] = 0;
  for (int i = tid; i < kWarps * S; i += kThreads) cnt[i] = 0;
  __syncthreads();
  // this CTA's choices, a consecutive part for each warp: counted here, ranked below
  const int n_flat = a.T * a.k;
  const int lo = c * a.chunk * a.k, count = min(n_flat - lo, a.chunk * a.k);
  const int part = ((count + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int wlo = min(count, warp * part), whi = min(count, wlo + part);
  for (int i = wlo + lane; i < whi; i += 32) {
    const int e = codes[i];
    if (e >= 0) atomicAdd(&cnt[warp * S + e], 1);
  }
  // the counts of all CTAs: a thread has one expert and every `rows`-th CTA, its loads independent
  const int rows = max(1, kThreads / E);
  const bool last = c == chunks - 1;
  float p_sum = 0.f;               // (the last CTA) of its expert's probabilities, over every `rows`-th CTA
  if (tid < rows * E) {
    const int e = tid % E;
    int all = 0, mine = 0;
#pragma unroll 8
    for (int i = tid / E; i < chunks; i += rows) {
      const int v = all_hist[i * E + e];
      if (last) p_sum += all_psum[i * E + e];
      all += v;
      mine += i < c ? v : 0;
    }
    if (all) atomicAdd(&total[e], all);
    if (mine) atomicAdd(&before[e], mine);
  }
  __syncthreads();
  if (warp == 0) {                 // exclusive prefix sums of the kept counts
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      const int n = e < E ? (a.capacity > 0 ? min(total[e], a.capacity) : total[e]) : 0;
      int s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += up;
      }
      if (e < E) first[e] = run + s - n;
      run += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) first[E] = run;
  }
  for (int e = kWarps - 1 - warp; e < E; e += kWarps) {      // (from the last warp on: the first one is busy); a lane per warp's count
    const int n = cnt[lane * S + e];
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    cnt[lane * S + e] = before[e] + sum - n;
  }
  __syncthreads();
  for (int i0 = wlo; i0 < whi; i0 += 32) {
    const int i = i0 + lane;
    const int e = i < whi ? codes[i] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int place = 0;
    if (e >= 0) place = cnt[warp * S + e] + rank;
    __syncwarp();
    if (e >= 0 && rank == 0) cnt[warp * S + e] += __popc(same);
    __syncwarp();
    if (i < whi) {
      int row = -1;
      if (e >= 0 && place < first[e + 1] - first[e]) {
        row = first[e] + place;
        a.rows[row] = lo + i;
      }
      a.slots[lo + i] = row;
    }
  }
  for (int r = first[E] + c * kThreads + tid; r < n_flat; r += chunks * kThreads) a.rows[r] = -1;
  if (last) {
    for (int e = tid; e <= E; e += kThreads) {
      a.offsets[e] = first[e];
      if (e < E) a.counts[e] = total[e];
    }
    float s = tid < rows * E ? static_cast<float>(total[tid % E]) * p_sum : 0.f;
    s = group_sum<32>(s, 0xffffffffu);
    if (lane == 0) aux_part[warp] = s;
    __syncthreads();
    if (warp == 0) {
      s = group_sum<32>(lane < kWarps ? aux_part[lane] : 0.f, 0xffffffffu);
      if (lane == 0) a.aux[0] = s * (static_cast<float>(E) / static_cast<float>(n_flat)) / static_cast<float>(a.T);
    }
  }
}

constexpr int plan_smem_ints(int E) { return 3 * E + 1 + kWarps * (E | 1) + kWarps; }

template <class T, int LANES, int VALS>
__global__ void __launch_bounds__(kThreads)
route_fwd_kernel(const T* __restrict__ logits, RouteArgs a, int single) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ int sm[];
  constexpr int GROUPS = kThreads / LANES;
  const int E = a.E, tid = threadIdx.x, lane = tid & 31, gl = tid & (LANES - 1), group = tid / LANES;
  const uint32_t mask = group_mask<LANES>(lane);
  int* hist = sm;                                         // [E]
  float* psum = reinterpret_cast<float*>(sm + E);         // [E]
  int* codes = sm + 2 * E;                                // [T k] with one CTA
  int* rest = codes + (single ? a.T * a.k : 0);
  float* part = reinterpret_cast<float*>(rest);           // [kWarps][E | 1]
  for (int e = tid; e < E; e += kThreads) hist[e] = 0;
  __syncthreads();
  float acc[VALS];
#pragma unroll
  for (int v = 0; v < VALS; ++v) acc[v] = 0.f;
  const int t0 = blockIdx.x * a.chunk, t1 = min(a.T, t0 + a.chunk);
  float next[VALS];      // the logits of the token after the one that is worked on
  auto fetch = [&](int t) {
#pragma unroll
    for (int v = 0; v < VALS; ++v) next[v] = t < t1 && v * LANES + gl < E ? load_logit(logits + t * a.ld + v * LANES + gl) : -INFINITY;
  };
  fetch(t0 + group);
  for (int t = t0 + group; t < t1; t += GROUPS) {
    float x[VALS];
    uint32_t key[VALS];
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      x[v] = next[v];
      key[v] = v * LANES + gl < E ? to_key(x[v]) : 0u;
    }
    fetch(t + GROUPS);
    uint32_t my_key = 0;
    int my_e = 0;
    if constexpr (sizeof(T) == 2) {      // 16 bits of key and, falling, 16 of index
#pragma unroll
      for (int v = 0; v < VALS; ++v) key[v] = key[v] ? (key[v] & 0xffff0000u) | (0xffffu - (v * LANES + gl)) : 0u;
    }
    int index[VALS];
#pragma unroll
    for (int v = 0; v < VALS; ++v) index[v] = v * LANES + gl;
    if constexpr (VALS <= 4) {           // falling keys; equal ones stay in the order of their indices
#pragma unroll
      for (int i = 1; i < VALS; ++i)
#pragma unroll
        for (int v = VALS - 1; v >= i; --v) {
          const bool swap = key[v] > key[v - 1];
          const uint32_t lo = swap ? key[v - 1] : key[v], hi = swap ? key[v] : key[v - 1];
          const int ilo = swap ? index[v - 1] : index[v], ihi = swap ? index[v] : index[v - 1];
          key[v] = lo;
          key[v - 1] = hi;
          index[v] = ilo;
          index[v - 1] = ihi;
        }
    }
    for (int j = 0; j < a.k; ++j) {
      uint32_t best = key[0];
      if constexpr (VALS > 4) {
#pragma unroll
        for (int v = 1; v < VALS; ++v) best = max(best, key[v]);
      }
      best = __reduce_max_sync(mask, best);
      int at = 0x7fffffff;
      if constexpr (sizeof(T) == 4) {
        if constexpr (VALS <= 4) {
          if (key[0] == best) at = index[0];
        } else {
#pragma unroll
          for (int v = VALS - 1; v >= 0; --v)
            if (key[v] == best) at = index[v];
        }
        at = __reduce_min_sync(mask, at);
      } else {
        at = 0xffff - static_cast<int>(best & 0xffffu);
      }
      if constexpr (VALS <= 4) {
        if (index[0] == at) {
#pragma unroll
          for (int v = 0; v + 1 < VALS; ++v) {
            key[v] = key[v + 1];
            index[v] = index[v + 1];
          }
          key[VALS - 1] = 0;
          index[VALS - 1] = -1;
        }
      } else {
#pragma unroll
        for (int v = 0; v < VALS; ++v)
          if (index[v] == at) key[v] = 0;
      }
      if (gl == j) { my_key = best; my_e = at; }
    }
    // the key of a bf16 value: its low bits as to_key leaves them
    if constexpr (sizeof(T) == 2) my_key = (my_key >> 31) ? my_key & 0xffff0000u : my_key | 0xffffu;
    const float top = from_key(__shfl_sync(mask, my_key, 0, LANES));
    const bool made = gl < a.k && my_key != kKeyMinusInf;
    const float ex = made ? expf(from_key(my_key) - top) : 0.f;
    const float sum = group_sum<LANES>(ex, mask);
    if (gl < a.k) {
      const int64_t i = static_cast<int64_t>(t) * a.k + gl;
      a.weights[i] = made ? ex / sum : 0.f;
      a.experts[i] = my_e;
      const int code = made ? my_e : -1;
      if (single) codes[i] = code;
      else a.slots[i] = code;
      if (made) atomicAdd(&hist[my_e], 1);
    }
    if (top != -INFINITY) {
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < VALS; ++v) {
        x[v] = expf(x[v] - top);
        s += x[v];
      }
      s = group_sum<LANES>(s, mask);
      const float r = 1.f / s;
#pragma unroll
      for (int v = 0; v < VALS; ++v) acc[v] += x[v] * r;
    }
  }
#pragma unroll
  for (int v = 0; v < VALS; ++v) {
    const int e = v * LANES + gl;
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) acc[v] += __shfl_xor_sync(0xffffffffu, acc[v], o);
    if (lane < LANES && e < E) part[(tid >> 5) * (E | 1) + e] = acc[v];
  }
  __syncthreads();
  for (int e = tid >> 5; e < E; e += kWarps) {      // a warp adds up the warps' sums of one expert
    const float s = group_sum<32>(part[lane * (E | 1) + e], 0xffffffffu);
    if (lane != 0) continue;
    if (single) {
      psum[e] = s;
    } else {
      a.psum[static_cast<int64_t>(blockIdx.x) * E + e] = s;
      a.hist[static_cast<int64_t>(blockIdx.x) * E + e] = hist[e];
    }
  }
  if (single) {
    __syncthreads();
    plan_rows(a, codes, hist, psum, 0, 1, rest);
  }
}

__global__ void __launch_bounds__(kThreads)
route_plan_kernel(RouteArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ int sm[];
  plan_rows(a, a.slots + static_cast<int64_t>(blockIdx.x) * a.chunk * a.k, a.hist, a.psum, blockIdx.x, gridDim.x, sm);
}

template <class T, int LANES, int VALS>
__global__ void __launch_bounds__(kBwdThreads)
route_bwd_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ weights, const int* __restrict__ experts,
                 const int* __restrict__ counts, const float* __restrict__ dweights, const float* __restrict__ daux,
                 T* __restrict__ dlogits, int n_tokens, int E, int k) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int GROUPS = kBwdThreads / LANES;
  const int tid = threadIdx.x, lane = tid & 31, gl = tid & (LANES - 1);
  const uint32_t mask = group_mask<LANES>(lane);
  const float pull = daux ? *daux * static_cast<float>(E) / static_cast<float>(n_tokens) : 0.f;
  const float per = 1.f / (static_cast<float>(n_tokens) * static_cast<float>(k));
  float share[VALS];
#pragma unroll
  for (int v = 0; v < VALS; ++v) share[v] = v * LANES + gl < E ? static_cast<float>(counts[v * LANES + gl]) * per : 0.f;
  for (int t = blockIdx.x * GROUPS + tid / LANES; t < n_tokens; t += gridDim.x * GROUPS) {
    float x[VALS], top = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      const int e = v * LANES + gl;
      x[v] = e < E ? load_logit(logits + t * ld + e) : -INFINITY;
      odd |= x[v] != x[v];
      top = fmaxf(top, x[v]);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o, LANES));
    odd = __any_sync(mask, odd);      // a NaN among the logits makes the whole row's gradient NaN
    if (odd) top = __uint_as_float(0x7fffffffu);
    float s = 0.f, mean = 0.f;
    const bool none = top == -INFINITY;
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      x[v] = none ? 0.f : expf(x[v] - top);
      s += x[v];
      mean += x[v] * share[v];
    }
    s = group_sum<LANES>(s, mask);
    mean = group_sum<LANES>(mean, mask);
    const float r = none ? 0.f : 1.f / s;
    mean *= r;
#pragma unroll
    for (int v = 0; v < VALS; ++v) x[v] = odd ? top : pull == 0.f ? 0.f : pull * (x[v] * r) * (share[v] - mean);
    if (dweights) {
      float w = 0.f, dw = 0.f;
      int e = -1;
      if (gl < k) {
        const int64_t i = static_cast<int64_t>(t) * k + gl;
        w = weights[i];
        e = experts[i];
        dw = w != 0.f ? dweights[i] : 0.f;
      }
      const float inner = group_sum<LANES>(w * dw, mask);
      const float g = w * (dw - inner);
      for (int j = 0; j < k; ++j) {
        const float gj = __shfl_sync(mask, g, j, LANES);
        const int ej = __shfl_sync(mask, e, j, LANES);
#pragma unroll
        for (int v = 0; v < VALS; ++v)
          if (ej == v * LANES + gl) x[v] += gj;
      }
    }
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      const int e = v * LANES + gl;
      if (e < E) dlogits[static_cast<int64_t>(t) * E + e] = static_cast<T>(x[v]);
    }
  }
}

int lanes_for(int E) {
  int l = 4;
  while (l < E && l < 32) l <<= 1;
  return l;
}

// (chunks, tokens of a chunk)
void chunks_for(int T, int E, int k, int& chunks, int& chunk) {
  const int groups = kThreads / lanes_for(E);
  // One CTA for as many tokens as it has groups.  One CTA, two kernels, us: 128 tokens x 8 experts 6.3, 7.5 and 256 tokens (two rounds) 8.2,
  // 7.5; 32 x 256 12.2, 13.8 and 64 (two rounds) 17.1, 13.8.
  if (T <= groups) {
    chunks = 1;
    chunk = T;
    return;
  }
  chunk = (T + kMaxChunks - 1) / kMaxChunks;
  chunk = (chunk + groups - 1) / groups * groups;
  chunks = (T + chunk - 1) / chunk;
}

#define TB_ROUTE_SIZES(CASE) CASE(4, 1) CASE(8, 1) CASE(16, 1) CASE(32, 1) CASE(32, 2) CASE(32, 4) CASE(32, 8) CASE(32, 16)

int vals_for(int E) {
  int v = 1;
  while (v * 32 < E) v <<= 1;
  return v;
}

template <class T>
int launch_fwd(const T* logits, const RouteArgs& a, int chunks, cudaStream_t stream) {
  const int lanes = lanes_for(a.E), vals = vals_for(a.E);
  const int plan = plan_smem_ints(a.E), sums = kWarps * (a.E | 1);
  const int smem = 4 * (chunks == 1 ? 2 * a.E + a.T * a.k + (sums > plan ? sums : plan) : 2 * a.E + sums);
#define CASE(L, V)                                                                                                            \
  if (lanes == L && vals == V) {                                                                                              \
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(route_fwd_kernel<T, L, V>), smem) ||                                \
        !ensure_dynamic_smem(reinterpret_cast<const void*>(route_plan_kernel), 4 * plan))                                      \
      return -20;                                                                                                             \
    int rc = launch_code(launch_pdl(route_fwd_kernel<T, L, V>, dim3(chunks), dim3(kThreads), smem, stream, logits, a, chunks == 1 ? 1 : 0)); \
    if (rc == 0 && chunks > 1)                                                                                                \
      rc = launch_code(launch_pdl(route_plan_kernel, dim3(chunks), dim3(kThreads), 4 * static_cast<size_t>(plan), stream, a)); \
    return rc;                                                                                                                \
  }
  TB_ROUTE_SIZES(CASE)
#undef CASE
  return -2;
}

}  // namespace

int64_t route_scratch_ints(int T, int E, int k) {
  int chunks, chunk;
  chunks_for(T, E, k, chunks, chunk);
  return 2 * static_cast<int64_t>(chunks) * E;
}

int route_kernels(int T, int E, int k) {
  int chunks, chunk;
  chunks_for(T, E, k, chunks, chunk);
  return chunks > 1 ? 2 : 1;
}

int route_fwd(const void* logits, bool bf16, int64_t ld, int T, int E, int k, int capacity, float* weights, int* experts, int* slots,
              int* offsets, int* rows, int* counts, float* aux, int* scratch, cudaStream_t stream) {
  if (T < 1 || E < 1 || E > kMaxExperts || k < 1 || k > E || k > kMaxChoices || static_cast<int64_t>(T) * k > (1ll << 30)) return -1;
  RouteArgs a{};
  a.ld = ld; a.T = T; a.E = E; a.k = k; a.capacity = capacity;
  a.weights = weights; a.experts = experts; a.slots = slots; a.offsets = offsets; a.rows = rows; a.counts = counts; a.aux = aux;
  int chunks;
  chunks_for(T, E, k, chunks, a.chunk);
  a.hist = scratch;
  a.psum = reinterpret_cast<float*>(scratch + static_cast<int64_t>(chunks) * E);
  return bf16 ? launch_fwd(static_cast<const __nv_bfloat16*>(logits), a, chunks, stream)
              : launch_fwd(static_cast<const float*>(logits), a, chunks, stream);
}

int route_bwd(const void* logits, bool bf16, int64_t ld, const float* weights, const int* experts, const int* counts,
              const float* dweights, const float* daux, void* dlogits, int T, int E, int k, cudaStream_t stream) {
  if (T < 1 || E < 1 || E > kMaxExperts || k < 1 || k > E || k > kMaxChoices) return -1;
  const int lanes = lanes_for(E), vals = vals_for(E);
  const int groups = kBwdThreads / lanes;
  const int need = (T + groups - 1) / groups;
  const int grid = need < 148 * 8 ? need : 148 * 8;
#define CASE(L, V)                                                                                                              \
  if (lanes == L && vals == V) {                                                                                                \
    const cudaError_t rc =                                                                                                      \
        bf16 ? launch_pdl(route_bwd_kernel<__nv_bfloat16, L, V>, dim3(grid), dim3(kBwdThreads), 0, stream,                          \
                          static_cast<const __nv_bfloat16*>(logits), ld, weights, experts, counts, dweights, daux,               \
                          static_cast<__nv_bfloat16*>(dlogits), T, E, k)                                                         \
             : launch_pdl(route_bwd_kernel<float, L, V>, dim3(grid), dim3(kBwdThreads), 0, stream,                                  \
                          static_cast<const float*>(logits), ld, weights, experts, counts, dweights, daux,                       \
                          static_cast<float*>(dlogits), T, E, k);                                                                \
    return launch_code(rc);                                                                                                      \
  }
  TB_ROUTE_SIZES(CASE)
#undef CASE
  return -2;
}

}  // namespace tb
