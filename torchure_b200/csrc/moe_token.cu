// The experts' feed-forward for one to four tokens without gradients, in two kernels: what the tokens' experts hold is read once, the
// sums are fp32 throughout, and between the two lies only the activation.
//
// Bound by the matrices (three per expert, 18.9 MB for two experts of 1024 x 1536) and, more so, by the chain router -> gate / up -> SwiGLU
// -> down -> weighted sum, a launch each on the way for more tokens.  Here every CTA of the first kernel finds the choices itself (a warp
// per token, about 1 us), and a warp computes gate and up of two units by reading four rows of the matrices; in the second kernel a
// warp computes one column of one token's output over all its experts.  Matrices are read past L1.  An expert that several tokens chose
// is read for each of them, from L2, which is why the kernels stop at four tokens.  One token, 2 of 8 experts of 1024 x 1536: 7.5 and 8.8 us
// from cold memory, 13 a call with the second kernel's launch under the first (2.9 us at copy bandwidth; the host takes 10.6).
#include "common.cuh"
#include "moe_api.h"

namespace tb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint4 load_once(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// sum of eight products
__device__ __forceinline__ float dot8(uint4 w, const float (&x)[8], float acc) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc = fmaf(__uint_as_float(u[i] << 16), x[2 * i], acc);
    acc = fmaf(__uint_as_float(u[i] & 0xffff0000u), x[2 * i + 1], acc);
  }
  return acc;
}
__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

struct Choices {
  int expert[kTokenChoices];       // -1: not made, or beyond the capacity
  float weight[kTokenChoices];
};

// The choices of all tokens, by the first T warps; everyone has them behind the caller's barrier.  With `aux`, the load-balancing term.
// Ties, closed experts and rows that are not finite: as in moe_route.cu.
template <int kVals, class L>      // kVals: logits of a lane
__device__ __forceinline__ void choose(const L* logits, int64_t ld, int T, int E, int k, int capacity, Choices* c, float* top_of, float* sum_of,
                                       float* aux) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < T) {
    float x[kVals];
    uint32_t key[kVals];
#pragma unroll
    for (int v = 0; v < kVals; ++v) {
      const int e = v * 32 + lane;
      x[v] = e < E ? load_logit(logits + warp * ld + e) : -INFINITY;
      const uint32_t u = __float_as_uint(x[v] + 0.f);
      key[v] = e >= E ? 0u : x[v] != x[v] ? 0xffffffffu : u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
    }
    float top = 0.f, mine = -INFINITY;
    int my_e = -1;
    for (int j = 0; j < k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int v = 0; v < kVals; ++v) best = max(best, key[v]);
      best = __reduce_max_sync(0xffffffffu, best);
      int at = 0x7fffffff;
#pragma unroll
      for (int v = kVals - 1; v >= 0; --v)
        if (key[v] == best) at = v * 32 + lane;
      at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
      for (int v = 0; v < kVals; ++v)
        if (at == v * 32 + lane) key[v] = 0;
      const float value = best == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float((best >> 31) ? best ^ 0x80000000u : ~best);
      if (j == 0) top = value;
      if (lane == j) { mine = value; my_e = at; }
    }
    const bool made = lane < k && mine != -INFINITY;
    const float ex = made ? expf(mine - top) : 0.f;
    const float sum = warp_sum(ex);
    if (lane < k) {
      c->expert[warp * k + lane] = made ? my_e : -1;
      c->weight[warp * k + lane] = made ? ex / sum : 0.f;
    }
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < kVals; ++v)
      if (v * 32 + lane < E) s += expf(x[v] - top);
    s = warp_sum(s);
    if (lane == 0) {
      top_of[warp] = top;
      sum_of[warp] = s;
    }
  }
  __syncthreads();
  const int n = T * k;
  if (aux && warp == 0) {
    // E sum_e share_e mean_t p[t, e], a choice at a time
    float s = 0.f;
    if (lane < n && c->expert[lane] >= 0)
      for (int t = 0; t < T; ++t)
        if (top_of[t] != -INFINITY) s += expf(load_logit(logits + t * ld + c->expert[lane]) - top_of[t]) / sum_of[t];
    s = warp_sum(s);
    if (lane == 0) *aux = s * static_cast<float>(E) / (static_cast<float>(n) * static_cast<float>(T));
  }
  if (capacity > 0) {
    int before = 0, e = -1;
    if (threadIdx.x < n) {
      e = c->expert[threadIdx.x];
      for (int i = 0; i < static_cast<int>(threadIdx.x); ++i) before += c->expert[i] == e;
    }
    __syncthreads();
    if (threadIdx.x < n && e >= 0 && before >= capacity) c->expert[threadIdx.x] = -1;
    __syncthreads();
  }
}

// h [T k, F] = silu(gate) up of every choice; choices and aux for the second kernel and the caller
template <int VALS, class L, class X>
__global__ void __launch_bounds__(kThreads)
token_up_kernel(const L* __restrict__ logits, int64_t ldl, const X* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ w,
                Choices* __restrict__ choices, float* __restrict__ h, float* __restrict__ aux, int T, int E, int k, int capacity, int D, int F) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ Choices c;
  __shared__ float top_of[kTokenTokens], sum_of[kTokenTokens];
  choose<VALS>(logits, ldl, T, E, k, capacity, &c, top_of, sum_of, blockIdx.x == 0 ? aux : nullptr);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = T * k;
  if (blockIdx.x == 0 && threadIdx.x < n) {
    choices->expert[threadIdx.x] = c.expert[threadIdx.x];
    choices->weight[threadIdx.x] = c.weight[threadIdx.x];
  }
  const int pairs = F / 2;
  for (int unit = blockIdx.x * kWarps + warp; unit < n * pairs; unit += gridDim.x * kWarps) {
    const int i = unit / pairs, f = unit % pairs * 2, e = c.expert[i];
    if (e < 0) continue;
    const __nv_bfloat16* gate = w + (static_cast<int64_t>(e) * 2 * F + f) * D;
    const __nv_bfloat16* up = gate + static_cast<int64_t>(F) * D;
    const X* row = x + (i / k) * ldx;
    float g0 = 0.f, g1 = 0.f, u0 = 0.f, u1 = 0.f;
#pragma unroll 4
    for (int d = lane * 8; d < D; d += 256) {
      const uint4 a = load_once(gate + d), b = load_once(gate + D + d), p = load_once(up + d), q = load_once(up + D + d);
      float v[8];
      load8(row + d, v);
      g0 = dot8(a, v, g0);
      g1 = dot8(b, v, g1);
      u0 = dot8(p, v, u0);
      u1 = dot8(q, v, u1);
    }
    // four sums over the warp: lanes 0 - 7 end up with the first, 8 - 15 with the second, ...
    const bool hi = lane & 16, mid = lane & 8;
    float s0 = (hi ? u0 : g0) + __shfl_xor_sync(0xffffffffu, hi ? g0 : u0, 16);
    float s1 = (hi ? u1 : g1) + __shfl_xor_sync(0xffffffffu, hi ? g1 : u1, 16);
    float s = (mid ? s1 : s0) + __shfl_xor_sync(0xffffffffu, mid ? s0 : s1, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float other = __shfl_xor_sync(0xffffffffu, s, 16);      // lanes 0 and 8: the up of their gate
    if (lane == 0 || lane == 8) h[static_cast<int64_t>(i) * F + f + (lane >> 3)] = s / (1.f + expf(-s)) * other;
  }
}

// out [T, D] = sum over a token's choices of weight times h W_down^T
template <class O>
__global__ void __launch_bounds__(kThreads)
token_down_kernel(const Choices* __restrict__ choices, const float* __restrict__ h, const __nv_bfloat16* __restrict__ w, O* __restrict__ out,
                  int T, int k, int D, int F) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ Choices c;
  if (threadIdx.x < T * k) {
    c.expert[threadIdx.x] = choices->expert[threadIdx.x];
    c.weight[threadIdx.x] = choices->weight[threadIdx.x];
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int unit = blockIdx.x * kWarps + warp; unit < T * D; unit += gridDim.x * kWarps) {
    const int t = unit / D, d = unit % D;
    float total = 0.f;
    for (int j0 = 0; j0 < k; j0 += 2) {      // two experts' rows at a time
      float sum[2] = {0.f, 0.f};
      const __nv_bfloat16* row[2];
      const float* act[2];
      bool in[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = t * k + j0 + j, e = j0 + j < k ? c.expert[i] : -1;
        in[j] = e >= 0;
        row[j] = w + (static_cast<int64_t>(in[j] ? e : 0) * D + d) * F;
        act[j] = h + static_cast<int64_t>(in[j] ? i : 0) * F;
      }
#pragma unroll 4
      for (int f = lane * 8; f < F; f += 256) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (in[j]) {
            const uint4 a = load_once(row[j] + f);
            float v[8];
            load8(act[j] + f, v);
            sum[j] = dot8(a, v, sum[j]);
          }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (in[j]) total = fmaf(c.weight[t * k + j0 + j], sum[j], total);
    }
    total = warp_sum(total);
    if (lane == 0) out[unit] = static_cast<O>(total);
  }
}

int grid_for(int64_t units) {
  const int64_t need = (units + kWarps - 1) / kWarps;
  return static_cast<int>(need < 148 * 4 ? need : 148 * 4);
}

}  // namespace

static_assert(kTokenChoices <= 32 && kTokenTokens <= kWarps, "a warp per token, a lane per choice");

int64_t token_scratch_bytes(int T, int k, int F) { return sizeof(Choices) + static_cast<int64_t>(T) * k * F * 4; }

int token_mlp(const void* logits, bool logits_bf16, int64_t ldl, const void* x, bool x_bf16, int64_t ldx, const __nv_bfloat16* w_gate_up,
              const __nv_bfloat16* w_down, void* out, float* aux, void* scratch, int T, int E, int k, int capacity, int D, int F,
              cudaStream_t stream) {
  if (T < 1 || T > kTokenTokens || k < 1 || k > E || T * k > kTokenChoices || E > kMaxExperts || D % 8 != 0 || F % 8 != 0 ||
      ldx % 8 != 0)
    return -1;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w_gate_up) | reinterpret_cast<uintptr_t>(w_down) |
        reinterpret_cast<uintptr_t>(scratch)) & 15) != 0)
    return -11;
  Choices* c = static_cast<Choices*>(scratch);
  float* h = reinterpret_cast<float*>(c + 1);
  static_assert(sizeof(Choices) % 16 == 0, "h on 16 bytes");
  const dim3 up(grid_for(static_cast<int64_t>(T) * k * (F / 2))), down(grid_for(static_cast<int64_t>(T) * D)), block(kThreads);
  cudaError_t rc;
  static_assert(kMaxExperts <= 12 * 32, "logits of a lane");
#define TB_UP_OF(V, L, X) \
  launch_pdl(token_up_kernel<V, L, X>, up, block, 0, stream, static_cast<const L*>(logits), ldl, static_cast<const X*>(x), ldx, w_gate_up, c, \
             h, aux, T, E, k, capacity, D, F)
#define TB_UP(L, X) (E <= 32 ? TB_UP_OF(1, L, X) : E <= 128 ? TB_UP_OF(4, L, X) : TB_UP_OF(12, L, X))
  if (logits_bf16) rc = x_bf16 ? TB_UP(__nv_bfloat16, __nv_bfloat16) : TB_UP(__nv_bfloat16, float);
  else rc = x_bf16 ? TB_UP(float, __nv_bfloat16) : TB_UP(float, float);
#undef TB_UP
#undef TB_UP_OF
  if (rc != cudaSuccess) return launch_code(rc);
  rc = x_bf16 ? launch_pdl(token_down_kernel<__nv_bfloat16>, down, block, 0, stream, c, h, w_down, static_cast<__nv_bfloat16*>(out), T, k, D, F)
              : launch_pdl(token_down_kernel<float>, down, block, 0, stream, c, h, w_down, static_cast<float*>(out), T, k, D, F);
  return launch_code(rc);
}

}  // namespace tb
