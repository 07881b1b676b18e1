// The router of a mixture of experts: top-k choice, weights, the order of rows by expert, the load-balancing term, and the
// gradient of weights and term; the same by scores, with a bias and groups of experts, and the bias' update.
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

// The k largest keys of a token, in falling order, the lowest index among equals: choice j in thread j of the token's (its key and index).  A
// thread's indices rise.  PACKED: a key carries its index in the low 16 bits, falling.
template <int VALS, bool PACKED>
__device__ __forceinline__ void choose(uint32_t (&key)[VALS], int (&index)[VALS], int k, int gl, uint32_t mask, uint32_t& my_key, int& my_e) {
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
  for (int j = 0; j < k; ++j) {
    uint32_t best = key[0];
    if constexpr (VALS > 4) {
#pragma unroll
      for (int v = 1; v < VALS; ++v) best = max(best, key[v]);
    }
    best = __reduce_max_sync(mask, best);
    int at = 0x7fffffff;
    if constexpr (!PACKED) {
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
}

// The same for threads of many keys, whose indices are not held: at(v) is that of key v.
template <int VALS, class At>
__device__ __forceinline__ void choose_wide(uint32_t (&key)[VALS], At at, int k, int gl, uint32_t mask, uint32_t& my_key, int& my_e) {
  for (int j = 0; j < k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int v = 1; v < VALS; ++v) best = max(best, key[v]);
    best = __reduce_max_sync(mask, best);
    int place = VALS;                // of this thread's lowest index with that key
#pragma unroll
    for (int v = VALS - 1; v >= 0; --v)
      if (key[v] == best) place = v;
    const int mine = place < VALS ? at(place) : 0x7fffffff, e = __reduce_min_sync(mask, mine);
    if (mine == e) {
#pragma unroll
      for (int v = 0; v < VALS; ++v)
        if (v == place) key[v] = 0;
    }
    if (gl == j) { my_key = best; my_e = e; }
  }
}

// What a CTA leaves of its tokens: the counts of its choices and the sums of its probabilities (those of each warp in `rest`, or a thread's in acc, of
// the experts `index`), or with one CTA the whole plan.
__device__ __forceinline__ void close_chunk(const RouteArgs& a, const int* codes, int* hist, float* psum, int* rest, int single) {
  const int E = a.E, tid = threadIdx.x, lane = tid & 31;
  const float* part = reinterpret_cast<const float*>(rest);           // [kWarps][E | 1]
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
template <int LANES, int VALS>
__device__ __forceinline__ void close_chunk(const RouteArgs& a, float (&acc)[VALS], const int (&index)[VALS], const int* codes, int* hist,
                                            float* psum, int* rest, int single) {
  const int E = a.E, tid = threadIdx.x, lane = tid & 31;
  float* part = reinterpret_cast<float*>(rest);           // [kWarps][E | 1]
#pragma unroll
  for (int v = 0; v < VALS; ++v) {
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) acc[v] += __shfl_xor_sync(0xffffffffu, acc[v], o);
    if (lane < LANES && index[v] < E) part[(tid >> 5) * (E | 1) + index[v]] = acc[v];
  }
  close_chunk(a, codes, hist, psum, rest, single);
}

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
  for (int e = tid; e < E; e += kThreads) hist[e] = 0;
  __syncthreads();
  float acc[VALS];
  int index[VALS];
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
#pragma unroll
    for (int v = 0; v < VALS; ++v) index[v] = v * LANES + gl;
    choose<VALS, sizeof(T) == 2>(key, index, a.k, gl, mask, my_key, my_e);
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
  for (int v = 0; v < VALS; ++v) index[v] = v * LANES + gl;
  close_chunk<LANES, VALS>(a, acc, index, codes, hist, psum, rest, single);
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

// ---- choice by scores, with a bias and groups of experts -----------------------------------------------
// s = sigmoid(l) or softmax(l), rounded to fp32 from 64 bits; with a bias or groups the choice goes by c = s + bias, else by l.  A group's score is
// the sum of its two largest c, or (group_scores 1) its largest; the experts of the top_groups largest groups stay open (ties to the lowest index).  Weights of the choices made:
//   w_j = scale s_j / (normalize: sum over the chosen of s_i, else 1);  aux = E sum_e share_e mean_t P[t, e], P = s / sum over all of s
// and with what = w / scale, d = 1 - s (sigmoid) or 1 (softmax):
//   dl_j += d_j what_j (scale dw_j - (normalize ? inner : 0)), inner = sum_i what_i scale dw_i;  softmax, not normalized: dl_e -= s_e inner
//   dl_e += daux E / T d_e P_e (share_e - sum_i share_i P_i)
// Scores 1e-7 apart decide which expert a token goes to and with it the order of all rows behind; computed in 32 bits they would depend on the
// machine's exp.  Rounded once from 64 they do so only within 2^-46 of the middle between two fp32 numbers: about one score in 2^22 may be the
// next number on another machine.
//
// Bound by instructions and latency, not by bytes (a score in 64 bits takes 33 instructions, a choice 25, and every token a warp).  32768 tokens x 128
// experts, 8 choices (8.4 MB of logits, 1.3 us): 32 us at 80 % of the issue slots, 780 instructions a token; 9 for the rows, 19 for the gradient at 57 %.
// 8192 x 256 in 8 groups, 8 choices: 25 us, 1.7 k instructions a token at 55 - 61 %: half of it issue, the rest waits for the token before (32 warps an
// SM, two rounds of tokens on 128 of them); 9 for the rows, 9 for the gradient (55 %).  One token 7.6.
struct ScoreArgs {
  const float* bias;       // nullptr: none
  int groups, top_groups, each;      // each: experts of a group
  int groups_log2;         // of the power of two that holds `groups`
  int sigmoid, normalize, group_scores;
  float scale;
};

// exp(-a) for a >= 0 in 64 bits, within about 2^-46: exp(-a) = 2^n exp(r), |r| <= ln 2 / 2, and Taylor's series to r^11 / 11!.  Above 700: what it is
// there, 2^-1010, next to which the result is zero in fp32.
__device__ __forceinline__ double exp_minus(float a) {
  const double x = static_cast<double>(fminf(a, 700.f));
  constexpr double kRound = 6755399441055744.0;      // 1.5 2^52: the sum's last bits are the rounded number
  const double t = fma(x, -1.4426950408889634, kRound);
  const double r = fma(t - kRound, -0.6931471805599453, -x);
  double p = 1.0 / 39916800.0;
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}
// sigmoid(l), rounded once to fp32: e = exp(-|l|), 1 / (1 + e) by two of Newton's steps
__device__ __forceinline__ float sigmoid64(float l) {
  const double e = exp_minus(fabsf(l)), d = 1.0 + e;
  double q = static_cast<double>(__fdividef(1.f, static_cast<float>(d)));
  q = fma(q, fma(-d, q, 1.0), q);
  q = fma(q, fma(-d, q, 1.0), q);
  const float s = static_cast<float>(l < 0.f ? e * q : q);
  return l != l ? l : s;
}
// s over exp(shift) for scores that may all be tiny: sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|))
__device__ __forceinline__ float sigmoid_over(float l, float shift) { return expf(fminf(l, 0.f) - shift) / (1.f + expf(-fabsf(l))); }
constexpr float kTinyScores = -80.f;      // a score below 2^-115: others may be too small for fp32

template <int LANES>
__device__ __forceinline__ float group_max(float v, uint32_t mask) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o, LANES));
  return v;
}
template <int LANES>
__device__ __forceinline__ double group_sum64(double v, uint32_t mask) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o, LANES);
  return v;
}

// The experts of a group lie with neighbouring threads: of the token's threads, LANES / 2^groups_log2 for each group.  Of more than eight experts a
// thread holds scores and keys only (1024 threads leave it 64 registers): sums lie in shared memory, the bias is read anew, the next token's logits are
// not on their way.  32768 tokens x 384 experts 107 us with the rows' numbers, 200 with all of it in registers; x 256, eight a thread, 81 and 70.
template <class T, int LANES, int VALS>
__global__ void __launch_bounds__(kThreads)
route_scored_kernel(const T* __restrict__ logits, RouteArgs a, ScoreArgs how, int single) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ int sm[];
  constexpr int GROUPS = kThreads / LANES;
  const int E = a.E, tid = threadIdx.x, lane = tid & 31, gl = tid & (LANES - 1), group = tid / LANES;
  const uint32_t mask = group_mask<LANES>(lane);
  const int per = LANES >> how.groups_log2, mine = gl / per, sub = gl - mine * per;      // threads of a group of experts, the group, the place in it
  int* hist = sm;                                         // [E]
  float* psum = reinterpret_cast<float*>(sm + E);         // [E]
  int* codes = sm + 2 * E;                                // [T k] with one CTA
  int* rest = codes + (single ? a.T * a.k : 0);
  for (int e = tid; e < E; e += kThreads) hist[e] = 0;
  __syncthreads();
  const bool by_score = how.bias != nullptr || how.groups > 1;
  constexpr bool kWide = VALS > 8;
  static_assert(!kWide || LANES == 32, "a warp's sums are a token's threads'");
  constexpr int kHeld = kWide ? 1 : VALS;
  const int here = mine < how.groups ? how.each : 0, first_expert = mine * how.each;
  const auto expert_at = [&](int v) { return v * per + sub < here ? first_expert + v * per + sub : 0x7fffffff; };
  float acc[kHeld], held_bias[kHeld];
  int held[kHeld];
  if constexpr (!kWide) {
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      held[v] = expert_at(v);
      acc[v] = 0.f;
      held_bias[v] = how.bias != nullptr && held[v] < E ? how.bias[held[v]] : 0.f;
    }
  }
  float* sums = reinterpret_cast<float*>(rest) + (tid >> 5) * (E | 1);      // (kWide) of this warp
  if constexpr (kWide) {
    for (int e = lane; e < E; e += 32) sums[e] = 0.f;
    __syncwarp();
  }
  const auto expert = [&](int v) {
    if constexpr (kWide) return expert_at(v);
    else return held[v];
  };
  const auto bias = [&](int v) {
    if constexpr (!kWide) return held_bias[v];
    else return how.bias != nullptr && expert_at(v) < E ? how.bias[expert_at(v)] : 0.f;
  };
  const auto gather = [&](float of, int v) {
    if constexpr (!kWide) acc[v] += of;
    else if (expert_at(v) < E) sums[expert_at(v)] += of;
  };
  const int t0 = blockIdx.x * a.chunk, t1 = min(a.T, t0 + a.chunk);
  float next[VALS];      // the logits of the token after the one that is worked on
  auto fetch = [&](int t) {
#pragma unroll
    for (int v = 0; v < VALS; ++v) next[v] = t < t1 && expert(v) < E ? load_logit(logits + t * a.ld + expert(v)) : -INFINITY;
  };
  if (!kWide) fetch(t0 + group);
  for (int t = t0 + group; t < t1; t += GROUPS) {
    float x[VALS], s[VALS], top = -INFINITY;
    if (kWide) fetch(t);
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      x[v] = next[v];
      top = fmaxf(top, x[v]);
    }
    if (!kWide) fetch(t + GROUPS);
    // (of sigmoids the largest logit is asked for only where all scores are tiny)
    const bool tiny = how.sigmoid && !__any_sync(mask, top >= kTinyScores);
    if (!how.sigmoid || tiny) top = group_max<LANES>(top, mask);
    if (how.sigmoid) {
#pragma unroll
      for (int v = 0; v < VALS; ++v) s[v] = sigmoid64(x[v]);
    } else {
      double e[VALS], sum = 0.0;
      const bool none = top == -INFINITY;
#pragma unroll
      for (int v = 0; v < VALS; ++v) {
        const float below = top - x[v];
        // (top passes NaN by: a row of -inf and NaN alone is not one without experts)
        e[v] = none ? (x[v] != x[v] ? static_cast<double>(x[v]) : 0.0) : below != below ? static_cast<double>(below) : exp_minus(below);
        sum += e[v];
      }
      sum = group_sum64<LANES>(sum, mask);
      const double r = none ? sum : 1.0 / sum;      // (none: 0, or NaN)
#pragma unroll
      for (int v = 0; v < VALS; ++v) s[v] = static_cast<float>(e[v] * r);
    }
    uint32_t key[VALS];
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      const float c = !by_score ? x[v] : x[v] == -INFINITY ? -INFINITY : s[v] + bias(v);
      key[v] = expert(v) < E ? to_key(c) : 0u;
    }
    if (how.groups > 1) {
      uint32_t first = 0, second = 0;      // the largest two of the group
#pragma unroll
      for (int v = 0; v < VALS; ++v) {
        second = max(second, min(first, key[v]));
        first = max(first, key[v]);
      }
      for (int o = per / 2; o > 0; o >>= 1) {
        const uint32_t f = __shfl_xor_sync(mask, first, o, LANES), g = __shfl_xor_sync(mask, second, o, LANES);
        second = max(max(second, g), min(first, f));
        first = max(first, f);
      }
      const uint32_t total = how.group_scores == 1 || second <= kKeyMinusInf ? first : to_key(from_key(first) + from_key(second));
      int ahead = 0;
      for (int g = 0; g < how.groups; ++g) {
        const uint32_t other = __shfl_sync(mask, total, g * per, LANES);
        ahead += other > total || (other == total && g < mine);
      }
      if (ahead >= how.top_groups) {
#pragma unroll
        for (int v = 0; v < VALS; ++v) key[v] = min(key[v], kKeyMinusInf);
      }
    }
    uint32_t my_key = 0;
    int my_e = 0;
    if constexpr (kWide) {
      choose_wide<VALS>(key, expert_at, a.k, gl, mask, my_key, my_e);
    } else {
      int index[VALS];
#pragma unroll
      for (int v = 0; v < VALS; ++v) index[v] = held[v];
      choose<VALS, false>(key, index, a.k, gl, mask, my_key, my_e);
    }
    const bool made = gl < a.k && my_key != kKeyMinusInf;
    const float l = made ? load_logit(logits + t * a.ld + my_e) : -INFINITY;
    float w = 0.f, whole = 1.f;
    if (how.sigmoid) {
      if (how.normalize && !__any_sync(mask, made && l >= kTinyScores)) {
        const float shift = group_max<LANES>(made ? l : -INFINITY, mask);
        if (made) w = sigmoid_over(l, fminf(shift, 0.f));
      } else if (made) {
        w = sigmoid64(l);
      }
      if (how.normalize) whole = group_sum<LANES>(w, mask);
    } else if (how.normalize) {
      const float shift = group_max<LANES>(l, mask);
      if (made) w = expf(l - shift);
      whole = group_sum<LANES>(w, mask);
    } else {
      if (made) w = expf(l - top);
      whole = 0.f;
#pragma unroll
      for (int v = 0; v < VALS; ++v) whole += top == -INFINITY ? 0.f : expf(x[v] - top);
      whole = group_sum<LANES>(whole, mask);
    }
    if (gl < a.k) {
      const int64_t i = static_cast<int64_t>(t) * a.k + gl;
      a.weights[i] = made ? how.scale * (w / whole) : 0.f;
      a.experts[i] = my_e;
      const int code = made ? my_e : -1;
      if (single) codes[i] = code;
      else a.slots[i] = code;
      if (made) atomicAdd(&hist[my_e], 1);
    }
    if (how.sigmoid) {
      if (tiny && top != -INFINITY) {      // over the largest one's
#pragma unroll
        for (int v = 0; v < VALS; ++v) s[v] = sigmoid_over(x[v], top);
      }
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < VALS; ++v) sum += s[v];
      sum = group_sum<LANES>(sum, mask);
      const float r = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int v = 0; v < VALS; ++v) gather(s[v] * r, v);
    } else {
#pragma unroll
      for (int v = 0; v < VALS; ++v) gather(s[v], v);
    }
  }
  if constexpr (kWide) close_chunk(a, codes, hist, psum, rest, single);
  else close_chunk<LANES, VALS>(a, acc, held, codes, hist, psum, rest, single);
}

template <class T, int LANES, int VALS>
__global__ void __launch_bounds__(kBwdThreads)
route_scored_bwd_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ weights, const int* __restrict__ experts,
                        const int* __restrict__ counts, const float* __restrict__ dweights, const float* __restrict__ daux,
                        T* __restrict__ dlogits, int n_tokens, int E, int k, int sigmoid, int normalize, float scale) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int GROUPS = kBwdThreads / LANES;
  const int tid = threadIdx.x, lane = tid & 31, gl = tid & (LANES - 1);
  const uint32_t mask = group_mask<LANES>(lane);
  const float pull = daux ? *daux * static_cast<float>(E) / static_cast<float>(n_tokens) : 0.f;
  const float per = 1.f / (static_cast<float>(n_tokens) * static_cast<float>(k));
  __shared__ float rows[GROUPS][LANES * VALS];
  float* row = rows[tid / LANES];
#pragma unroll
  for (int v = 0; v < VALS; ++v) row[v * LANES + gl] = 0.f;
  __syncwarp(mask);
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
    top = group_max<LANES>(top, mask);
    odd = __any_sync(mask, odd);      // a NaN among the logits makes the whole row's gradient NaN
    const bool none = top == -INFINITY;
    float p[VALS], steep[VALS], s = 0.f, mean = 0.f;
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      if (sigmoid) {
        const float e = expf(-fabsf(x[v])), q = __fdividef(1.f, 1.f + e);
        p[v] = x[v] < 0.f ? e * q : q;
        steep[v] = x[v] < 0.f ? q : e * q;
        if (top < kTinyScores) p[v] = none ? 0.f : sigmoid_over(x[v], top);
      } else {
        p[v] = none ? 0.f : expf(x[v] - top);
      }
      s += p[v];
      mean += p[v] * share[v];
    }
    s = group_sum<LANES>(s, mask);
    mean = group_sum<LANES>(mean, mask);
    const float r = none ? 0.f : 1.f / s;
    mean *= r;
    float w = 0.f, dw = 0.f, inner = 0.f, g = 0.f;
    int e_j = -1;
    if (dweights) {
      if (gl < k) {
        const int64_t i = static_cast<int64_t>(t) * k + gl;
        w = weights[i] / scale;
        e_j = experts[i];
        dw = w != 0.f ? scale * dweights[i] : 0.f;
      }
      inner = group_sum<LANES>(w * dw, mask);
      g = w * (dw - (normalize ? inner : 0.f));
      // (an expert of a choice that was not made may have any logit)
      if (sigmoid && g != 0.f && e_j >= 0 && e_j < E) g *= sigmoid_over(-load_logit(logits + t * ld + e_j), 0.f);
      if (normalize || sigmoid) inner = 0.f;      // from here on what every expert pays for a softmax's sum
    }
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      const float q = p[v] * r;
      float d = pull == 0.f ? 0.f : pull * q * (share[v] - mean);
      if (sigmoid) d *= steep[v];
      else d -= q * inner;
      x[v] = odd ? __uint_as_float(0x7fffffffu) : d;
    }
    if (dweights) {      // each choice's share to its expert's thread, through the token's row in shared memory
      const bool gives = e_j >= 0 && e_j < E;
      if (gives) row[e_j] = g;
      __syncwarp(mask);
#pragma unroll
      for (int v = 0; v < VALS; ++v) x[v] += row[v * LANES + gl];
      __syncwarp(mask);
      if (gives) row[e_j] = 0.f;
      __syncwarp(mask);
    }
#pragma unroll
    for (int v = 0; v < VALS; ++v) {
      const int e = v * LANES + gl;
      if (e < E) dlogits[static_cast<int64_t>(t) * E + e] = static_cast<T>(x[v]);
    }
  }
}

// bias[e] += rate sign(mean of the counts - counts[e]), the comparison in whole numbers
__global__ void __launch_bounds__(kThreads)
balance_bias_kernel(float* __restrict__ bias, const int* __restrict__ counts, int E, float rate) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ long long parts[kWarps];
  const int tid = threadIdx.x, lane = tid & 31;
  long long sum = 0;
  for (int e = tid; e < E; e += kThreads) sum += counts[e];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) parts[tid >> 5] = sum;
  __syncthreads();
  sum = parts[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  for (int e = tid; e < E; e += kThreads) {
    const long long over = static_cast<long long>(counts[e]) * E - sum;
    bias[e] += over < 0 ? rate : over > 0 ? -rate : 0.f;
  }
}

int lanes_for(int E) {
  int l = 4;
  while (l < E && l < 32) l <<= 1;
  return l;
}

// (chunks, tokens of a chunk)
void chunks_for(int T, int lanes, int& chunks, int& chunk) {
  const int groups = kThreads / lanes;
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

bool score_fits(int E, int k, const RouteScore& how) {
  return how.groups >= 1 && how.groups <= kMaxExpertGroups && E % how.groups == 0 && how.top_groups >= 1 && how.top_groups <= how.groups &&
         (how.group_scores == 1 || how.group_scores == 2) && k <= how.top_groups * (E / how.groups);
}

// Threads of a token, logits of a thread and log2 of the groups' places: each group has the same power of two of threads.
void scored_shape(int E, const RouteScore& how, int& lanes, int& vals, int& groups_log2) {
  groups_log2 = 0;
  while ((1 << groups_log2) < how.groups) ++groups_log2;
  const int each = E / how.groups;
  lanes = 4;
  while (lanes < 32 && (lanes >> groups_log2) < each) lanes <<= 1;
  vals = 1;
  while (vals * (lanes >> groups_log2) < each) vals = vals < 8 ? vals * 2 : vals + (vals < 16 ? 4 : 8);
}

int lanes_of(int E, const RouteScore* how) {
  if (how == nullptr) return lanes_for(E);
  int lanes, vals, log2;
  scored_shape(E, *how, lanes, vals, log2);
  return lanes;
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

// (groups that are no power of two leave threads without experts: up to 22 logits for the others)
#define TB_SCORED_SIZES(CASE) CASE(4, 1) CASE(8, 1) CASE(16, 1) CASE(32, 1) CASE(32, 2) CASE(32, 4) CASE(32, 8) CASE(32, 12) CASE(32, 16) CASE(32, 24)

template <class T>
int launch_scored(const T* logits, const RouteArgs& a, const RouteScore& how, int chunks, cudaStream_t stream) {
  int lanes, vals;
  ScoreArgs s{};
  scored_shape(a.E, how, lanes, vals, s.groups_log2);
  s.bias = how.bias; s.groups = how.groups; s.top_groups = how.top_groups; s.each = a.E / how.groups;
  s.sigmoid = how.sigmoid; s.normalize = how.normalize; s.scale = how.scale; s.group_scores = how.group_scores;
  const int plan = plan_smem_ints(a.E), sums = kWarps * (a.E | 1);
  const int smem = 4 * (chunks == 1 ? 2 * a.E + a.T * a.k + (sums > plan ? sums : plan) : 2 * a.E + sums);
#define CASE(L, V)                                                                                                                 \
  if (lanes == L && vals == V) {                                                                                                   \
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(route_scored_kernel<T, L, V>), smem) ||                                  \
        !ensure_dynamic_smem(reinterpret_cast<const void*>(route_plan_kernel), 4 * plan))                                           \
      return -20;                                                                                                                  \
    int rc = launch_code(                                                                                                          \
        launch_pdl(route_scored_kernel<T, L, V>, dim3(chunks), dim3(kThreads), smem, stream, logits, a, s, chunks == 1 ? 1 : 0));     \
    if (rc == 0 && chunks > 1)                                                                                                     \
      rc = launch_code(launch_pdl(route_plan_kernel, dim3(chunks), dim3(kThreads), 4 * static_cast<size_t>(plan), stream, a));      \
    return rc;                                                                                                                     \
  }
  TB_SCORED_SIZES(CASE)
#undef CASE
  return -2;
}

}  // namespace

int balance_bias(float* bias, const int* counts, int E, float rate, cudaStream_t stream) {
  if (E < 1) return -1;
  return launch_code(launch_pdl(balance_bias_kernel, dim3(1), dim3(kThreads), 0, stream, bias, counts, E, rate));
}

int64_t route_scratch_ints(int T, int E, const RouteScore* how) {
  int chunks, chunk;
  chunks_for(T, lanes_of(E, how), chunks, chunk);
  return 2 * static_cast<int64_t>(chunks) * E;
}

int route_kernels(int T, int E, const RouteScore* how) {
  int chunks, chunk;
  chunks_for(T, lanes_of(E, how), chunks, chunk);
  return chunks > 1 ? 2 : 1;
}

int route_fwd(const void* logits, bool bf16, int64_t ld, int T, int E, int k, int capacity, const RouteScore* how, float* weights,
              int* experts, int* slots, int* offsets, int* rows, int* counts, float* aux, int* scratch, cudaStream_t stream) {
  if (T < 1 || E < 1 || E > kMaxExperts || k < 1 || k > E || k > kMaxChoices || static_cast<int64_t>(T) * k > (1ll << 30)) return -1;
  if (how != nullptr && !score_fits(E, k, *how)) return -1;
  RouteArgs a{};
  a.ld = ld; a.T = T; a.E = E; a.k = k; a.capacity = capacity;
  a.weights = weights; a.experts = experts; a.slots = slots; a.offsets = offsets; a.rows = rows; a.counts = counts; a.aux = aux;
  int chunks;
  chunks_for(T, lanes_of(E, how), chunks, a.chunk);
  a.hist = scratch;
  a.psum = reinterpret_cast<float*>(scratch + static_cast<int64_t>(chunks) * E);
  if (how != nullptr)
    return bf16 ? launch_scored(static_cast<const __nv_bfloat16*>(logits), a, *how, chunks, stream)
                : launch_scored(static_cast<const float*>(logits), a, *how, chunks, stream);
  return bf16 ? launch_fwd(static_cast<const __nv_bfloat16*>(logits), a, chunks, stream)
              : launch_fwd(static_cast<const float*>(logits), a, chunks, stream);
}

int route_bwd(const void* logits, bool bf16, int64_t ld, const float* weights, const int* experts, const int* counts,
              const float* dweights, const float* daux, void* dlogits, int T, int E, int k, const RouteScore* how, cudaStream_t stream) {
  if (T < 1 || E < 1 || E > kMaxExperts || k < 1 || k > E || k > kMaxChoices) return -1;
  if (how != nullptr && !score_fits(E, k, *how)) return -1;
  const int lanes = lanes_for(E), vals = vals_for(E);
  const int groups = kBwdThreads / lanes;
  const int need = (T + groups - 1) / groups;
  const int grid = need < 148 * 8 ? need : 148 * 8;
  if (how != nullptr) {
#define CASE(L, V)                                                                                                              \
  if (lanes == L && vals == V) {                                                                                                \
    const cudaError_t rc =                                                                                                      \
        bf16 ? launch_pdl(route_scored_bwd_kernel<__nv_bfloat16, L, V>, dim3(grid), dim3(kBwdThreads), 0, stream,                  \
                          static_cast<const __nv_bfloat16*>(logits), ld, weights, experts, counts, dweights, daux,               \
                          static_cast<__nv_bfloat16*>(dlogits), T, E, k, how->sigmoid ? 1 : 0, how->normalize ? 1 : 0, how->scale) \
             : launch_pdl(route_scored_bwd_kernel<float, L, V>, dim3(grid), dim3(kBwdThreads), 0, stream,                          \
                          static_cast<const float*>(logits), ld, weights, experts, counts, dweights, daux,                       \
                          static_cast<float*>(dlogits), T, E, k, how->sigmoid ? 1 : 0, how->normalize ? 1 : 0, how->scale);        \
    return launch_code(rc);                                                                                                      \
  }
  TB_ROUTE_SIZES(CASE)
#undef CASE
    return -2;
  }
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
