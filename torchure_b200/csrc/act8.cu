// Activation checkpoints in 8 bits: quantised as they are written, and read by the backward pass of SwiGLU.
//
// A row is cut into blocks of 64 values.  With a the block's largest magnitude, q = sign(x) floor(127 |x| / a + 1/2) and scale =
// a / 127; what is kept stands for q scale, off by a / 254 at most.  A block of zeros has scale 0; one that holds a NaN or an infinity
// has scale NaN, so that it reads back as NaN instead of as numbers.
//
// x has 8 significant bits, so 127 |x| / a is either exactly half-way between two whole numbers or at least 2^-17 (relative) away
// from it.  The product with 127 / a, raised by 2^-20, therefore rounds to the nearest whole number as the quotient does, and
// half-way cases away from zero, without a division per value.
//
// Bound by memory.  Eight lanes have a block, eight values each (16 bytes of bf16, 8 bytes of int8); widths that are no multiple of
// 8, or rows off a 16-byte boundary, are read value by value.
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

template <bool VEC>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int left, float (&v)[8]) {
  if (VEC) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (left > 0) u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? __bfloat162float(p[i]) : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(__nv_bfloat16* p, int left, const float (&v)[8]) {
  if (VEC) {
    if (left > 0)
      *reinterpret_cast<uint4*>(p) =
          make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = __float2bfloat16(v[i]);
  }
}
template <bool VEC>
__device__ __forceinline__ void load_q(const int8_t* p, int left, float scale, float (&v)[8]) {
  if (VEC) {
    int2 u = make_int2(0, 0);
    if (left > 0) u = *reinterpret_cast<const int2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = static_cast<float>(static_cast<int8_t>(u.x >> (8 * i))) * scale;
      v[4 + i] = static_cast<float>(static_cast<int8_t>(u.y >> (8 * i))) * scale;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? static_cast<float>(p[i]) * scale : 0.f;
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {      // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The block of this thread's group of eight lanes: 8 values each, `left` of them inside the row.
template <bool VEC>
__device__ __forceinline__ void keep8(const float (&v)[8], int left, int8_t* q, float* scale, bool first) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max_nan(a, fabsf(v[i]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  const bool finite = a <= 3.4028235e38f;
  // 127 / a is no float for the smallest a: such blocks count as zeros, off by less than 2^-120
  const bool some = finite && a >= 7.52316385e-37f;
  const float inv = some ? __fdiv_rn(127.f, a) * 1.00000095367431640625f : 0.f;
  if (first) *scale = finite ? (some ? __fdiv_rn(a, 127.f) : 0.f) : __uint_as_float(0x7fffffffu);
  int w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = some ? __float2int_rn(v[i] * inv) : 0;
  if (VEC) {
    if (left > 0) {
      int2 u = make_int2(0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u.x |= (w[i] & 0xff) << (8 * i);
        u.y |= (w[4 + i] & 0xff) << (8 * i);
      }
      *reinterpret_cast<int2*>(q) = u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) q[i] = static_cast<int8_t>(w[i]);
  }
}

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// units: blocks of a matrix; a block is worked on by eight lanes
template <bool VEC>
__global__ void __launch_bounds__(kThreads)
quantize8_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, float* __restrict__ scales, int64_t M, int N,
                 int nb) {
  pdl_wait();
  pdl_launch_dependents();
  const int g = threadIdx.x & 7;
  const int64_t units = M * nb, step = static_cast<int64_t>(gridDim.x) * (kThreads / 8);
  for (int64_t u0 = static_cast<int64_t>(blockIdx.x) * (kThreads / 8) + (threadIdx.x >> 5) * 4; u0 < units; u0 += step) {
    const int64_t u = u0 + ((threadIdx.x & 31) >> 3);      // whole warps stay: the lanes of a block shuffle
    const bool in = u < units;
    const int64_t row = in ? u / nb : 0;
    const int b = in ? static_cast<int>(u - row * nb) : 0, c = b * kActBlock + g * 8;
    const int left = in ? N - c : 0;
    float v[8];
    load8<VEC>(x + row * ldx + c, left, v);
    keep8<VEC>(v, left, q + row * N + c, scales + row * nb + b, in && g == 0);
  }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads)
dequantize8_kernel(const int8_t* __restrict__ q, const float* __restrict__ scales, __nv_bfloat16* __restrict__ x, int64_t M, int N,
                   int nb) {
  pdl_wait();
  pdl_launch_dependents();
  const int g = threadIdx.x & 7;
  const int64_t units = M * nb, step = static_cast<int64_t>(gridDim.x) * (kThreads / 8);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kThreads / 8) + (threadIdx.x >> 3); u < units; u += step) {
    const int64_t row = u / nb;
    const int b = static_cast<int>(u - row * nb), c = b * kActBlock + g * 8;
    float v[8];
    load_q<VEC>(q + row * N + c, N - c, scales[u], v);
    store8<VEC>(x + row * N + c, N - c, v);
  }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads)
swiglu8_fwd_kernel(const __nv_bfloat16* __restrict__ gu, int64_t ldgu, __nv_bfloat16* __restrict__ act, int8_t* __restrict__ q,
                   float* __restrict__ scales, int64_t M, int F, int nb) {
  pdl_wait();
  pdl_launch_dependents();
  const int lg = threadIdx.x & 7;
  const int64_t units = M * nb, step = static_cast<int64_t>(gridDim.x) * (kThreads / 8);
  for (int64_t u0 = static_cast<int64_t>(blockIdx.x) * (kThreads / 8) + (threadIdx.x >> 5) * 4; u0 < units; u0 += step) {
    const int64_t u = u0 + ((threadIdx.x & 31) >> 3);
    const bool in = u < units;
    const int64_t row = in ? u / nb : 0;
    const int b = in ? static_cast<int>(u - row * nb) : 0, c = b * kActBlock + lg * 8;
    const int left = in ? F - c : 0;
    float gate[8], up[8], out[8];
    load8<VEC>(gu + row * ldgu + c, left, gate);
    load8<VEC>(gu + row * ldgu + F + c, left, up);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = gate[i] * sigmoid(gate[i]) * up[i];
    store8<VEC>(act + row * F + c, left, out);
    keep8<VEC>(gate, left, q + row * 2 * F + c, scales + row * 2 * nb + b, in && lg == 0);
    keep8<VEC>(up, left, q + row * 2 * F + F + c, scales + row * 2 * nb + nb + b, in && lg == 0);
  }
}

// d silu(g) u of gate and up, given d(act)
__device__ __forceinline__ void swiglu_grad(const float (&g)[8], const float (&u)[8], const float (&d)[8], float (&dg)[8], float (&du)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = sigmoid(g[i]);
    dg[i] = d[i] * u[i] * s * (1.f + g[i] * (1.f - s));
    du[i] = d[i] * g[i] * s;
  }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads)
swiglu8_bwd_kernel(const __nv_bfloat16* __restrict__ dact, int64_t ldd, const int8_t* __restrict__ q, const float* __restrict__ scales,
                   __nv_bfloat16* __restrict__ dgu, int64_t M, int F, int nb) {
  pdl_wait();
  pdl_launch_dependents();
  const int lg = threadIdx.x & 7;
  const int64_t units = M * nb, step = static_cast<int64_t>(gridDim.x) * (kThreads / 8);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kThreads / 8) + (threadIdx.x >> 3); u < units; u += step) {
    const int64_t row = u / nb;
    const int b = static_cast<int>(u - row * nb), c = b * kActBlock + lg * 8, left = F - c;
    float gate[8], up[8], d[8], dg[8], du[8];
    load_q<VEC>(q + row * 2 * F + c, left, scales[row * 2 * nb + b], gate);
    load_q<VEC>(q + row * 2 * F + F + c, left, scales[row * 2 * nb + nb + b], up);
    load8<VEC>(dact + row * ldd + c, left, d);
    swiglu_grad(gate, up, d, dg, du);
    store8<VEC>(dgu + row * 2 * F + c, left, dg);
    store8<VEC>(dgu + row * 2 * F + F + c, left, du);
  }
}

// One warp per choice: the row of its gradient and the dot product that is its weight's.
template <bool Q8, bool VEC>
__global__ void __launch_bounds__(kThreads)
expert_swiglu_bwd_kernel(const __nv_bfloat16* __restrict__ s, const __nv_bfloat16* __restrict__ gu, const int8_t* __restrict__ q,
                         const float* __restrict__ scales, const float* __restrict__ weights, const int* __restrict__ slots,
                         const int* __restrict__ offsets, __nv_bfloat16* __restrict__ dgu, __nv_bfloat16* __restrict__ act_w,
                         float* __restrict__ dweights, int R, int E, int F, int nb) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int live = min(max(offsets[E], 0), R);
  for (int i = blockIdx.x * kWarps + (threadIdx.x >> 5); i < R; i += gridDim.x * kWarps) {
    const int r = slots[i];
    float dot = 0.f;
    if (r >= 0 && r < R) {
      const float w = weights[i];
      const int64_t row = r;
      for (int c = lane * 8; c < F; c += 256) {
        const int left = F - c;
        float gate[8], up[8], d[8], dg[8], du[8], a[8];
        if (Q8) {
          load_q<VEC>(q + row * 2 * F + c, left, scales[row * 2 * nb + c / kActBlock], gate);
          load_q<VEC>(q + row * 2 * F + F + c, left, scales[row * 2 * nb + nb + c / kActBlock], up);
        } else {
          load8<VEC>(gu + row * 2 * F + c, left, gate);
          load8<VEC>(gu + row * 2 * F + F + c, left, up);
        }
        load8<VEC>(s + row * F + c, left, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a[j] = gate[j] * sigmoid(gate[j]) * up[j];
          dot = fmaf(a[j], d[j], dot);
          a[j] *= w;
          d[j] *= w;
        }
        swiglu_grad(gate, up, d, dg, du);
        store8<VEC>(act_w + row * F + c, left, a);
        store8<VEC>(dgu + row * 2 * F + c, left, dg);
        store8<VEC>(dgu + row * 2 * F + F + c, left, du);
      }
      dot = warp_sum(dot);
    }
    if (lane == 0) dweights[i] = dot;
    if (i >= live) {      // row i is no choice's
      const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int c = lane * 8; c < F; c += 256) {
        store8<VEC>(act_w + static_cast<int64_t>(i) * F + c, F - c, zero);
        store8<VEC>(dgu + static_cast<int64_t>(i) * 2 * F + c, F - c, zero);
        store8<VEC>(dgu + static_cast<int64_t>(i) * 2 * F + F + c, F - c, zero);
      }
    }
  }
}

int blocks_of(int n) { return (n + kActBlock - 1) / kActBlock; }
int grid_for(int64_t units, int per_cta) {
  const int64_t need = (units + per_cta - 1) / per_cta;
  return static_cast<int>(need < 148 * 16 ? need : 148 * 16);
}
bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

void quantize8(const __nv_bfloat16* x, int64_t ldx, int8_t* q, float* scales, int64_t M, int N, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return;
  const int nb = blocks_of(N);
  const dim3 grid(grid_for(M * nb, kThreads / 8)), block(kThreads);
  if (N % 8 == 0 && ldx % 8 == 0 && at16(x) && at16(q)) launch_pdl(quantize8_kernel<true>, grid, block, 0, stream, x, ldx, q, scales, M, N, nb);
  else launch_pdl(quantize8_kernel<false>, grid, block, 0, stream, x, ldx, q, scales, M, N, nb);
}

void dequantize8(const int8_t* q, const float* scales, __nv_bfloat16* x, int64_t M, int N, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return;
  const int nb = blocks_of(N);
  const dim3 grid(grid_for(M * nb, kThreads / 8)), block(kThreads);
  if (N % 8 == 0 && at16(x) && at16(q)) launch_pdl(dequantize8_kernel<true>, grid, block, 0, stream, q, scales, x, M, N, nb);
  else launch_pdl(dequantize8_kernel<false>, grid, block, 0, stream, q, scales, x, M, N, nb);
}

void swiglu8_fwd(const __nv_bfloat16* gu, int64_t ldgu, __nv_bfloat16* act, int8_t* q, float* scales, int64_t M, int F,
                 cudaStream_t stream) {
  if (M <= 0 || F <= 0) return;
  const int nb = blocks_of(F);
  const dim3 grid(grid_for(M * nb, kThreads / 8)), block(kThreads);
  if (F % 8 == 0 && ldgu % 8 == 0 && at16(gu) && at16(act) && at16(q))
    launch_pdl(swiglu8_fwd_kernel<true>, grid, block, 0, stream, gu, ldgu, act, q, scales, M, F, nb);
  else launch_pdl(swiglu8_fwd_kernel<false>, grid, block, 0, stream, gu, ldgu, act, q, scales, M, F, nb);
}

void swiglu8_bwd(const __nv_bfloat16* dact, int64_t ldd, const int8_t* q, const float* scales, __nv_bfloat16* dgu, int64_t M, int F,
                 cudaStream_t stream) {
  if (M <= 0 || F <= 0) return;
  const int nb = blocks_of(F);
  const dim3 grid(grid_for(M * nb, kThreads / 8)), block(kThreads);
  if (F % 8 == 0 && ldd % 8 == 0 && at16(dact) && at16(dgu) && at16(q))
    launch_pdl(swiglu8_bwd_kernel<true>, grid, block, 0, stream, dact, ldd, q, scales, dgu, M, F, nb);
  else launch_pdl(swiglu8_bwd_kernel<false>, grid, block, 0, stream, dact, ldd, q, scales, dgu, M, F, nb);
}

void expert_swiglu_bwd(const __nv_bfloat16* s, const __nv_bfloat16* gu, const int8_t* q, const float* scales, const float* weights,
                       const int* slots, const int* offsets, __nv_bfloat16* dgu, __nv_bfloat16* act_w, float* dweights, int R, int E,
                       int F, cudaStream_t stream) {
  if (R <= 0 || F <= 0) return;
  const int nb = blocks_of(F);
  const dim3 grid(grid_for(R, kWarps)), block(kThreads);
  const bool vec = F % 8 == 0 && at16(s) && at16(dgu) && at16(act_w) && (gu ? at16(gu) : at16(q));
#define TB_EXPERT(Q, V) \
  launch_pdl(expert_swiglu_bwd_kernel<Q, V>, grid, block, 0, stream, s, gu, q, scales, weights, slots, offsets, dgu, act_w, dweights, R, E, F, nb)
  if (gu) { if (vec) TB_EXPERT(false, true); else TB_EXPERT(false, false); }
  else { if (vec) TB_EXPERT(true, true); else TB_EXPERT(true, false); }
#undef TB_EXPERT
}

}  // namespace tb
