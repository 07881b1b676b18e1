// Activation checkpoints in 8 bits: quantised as they are written, and read by the backward pass of SwiGLU.
//
// A row is cut into blocks of 64 values.  With a the block's largest magnitude, q = sign(x) floor(127 |x| / a + 1/2) and scale =
// a / 127; what is kept stands for q scale, off by a / 254 at most.  A block of zeros has scale 0; one that holds a NaN or an infinity
// has scale NaN, so that it reads back as NaN instead of as numbers.
//
// x has 8 significant bits, so 127 |x| / a is either exactly half-way between two whole numbers or at least 2^-17 (relative) away
// from it.  The product with 127 / a, raised by 2^-20, therefore rounds to the nearest whole number as the quotient does, and
// half-way cases away from zero, without a division per value; 127 / a itself may be off by 2^-21.
//
// The arithmetic has to stay below the memory's time: the largest magnitude is found on packed bf16 pairs, whole numbers are taken
// from the low byte of x (127 / a) + 1.5 2^23 and put together by byte permutations, and read back the other way (conversion
// instructions run at a quarter of the rate).
//
// Bound by memory.  Eight lanes have a block, eight values each (16 bytes of bf16, 8 bytes of int8), four blocks at a time (SwiGLU:
// two of gate and two of up) so that as many loads are on their way; with one block at a time 16384 x 2560 took 43 us to quantise and
// 32 to read back, and SwiGLU of 16384 x 1536 54 and 42.  Widths that are no multiple of 8, or rows off a 16-byte boundary, are read
// value by value.
#include "act8.cuh"
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

// 8 bf16 values as they lie, `left` of them inside the row, zeros behind
template <bool VEC>
__device__ __forceinline__ uint4 load_raw(const __nv_bfloat16* p, int left) {
  if (VEC) return left > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
  uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) u[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void spread(uint4 raw, float (&v)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int left, float (&v)[8]) { spread(load_raw<VEC>(p, left), v); }
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
// 8 kept values as they lie
template <bool VEC>
__device__ __forceinline__ uint2 load_q(const int8_t* p, int left) {
  if (VEC) return left > 0 ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
  uint32_t u[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) u[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(p[i])) << (8 * (i & 3));
  return make_uint2(u[0], u[1]);
}
// what they stand for: byte b ^ 128 under the exponent of 2^23 is 2^23 + 128 + b
__device__ __forceinline__ void read_q(uint2 raw, float scale, float (&v)[8]) {
  const uint32_t w[2] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = (__uint_as_float(__byte_perm(w[i], 0x4b000000u, 0x7650)) - 8388736.f) * scale;
    v[4 * i + 1] = (__uint_as_float(__byte_perm(w[i], 0x4b000000u, 0x7651)) - 8388736.f) * scale;
    v[4 * i + 2] = (__uint_as_float(__byte_perm(w[i], 0x4b000000u, 0x7652)) - 8388736.f) * scale;
    v[4 * i + 3] = (__uint_as_float(__byte_perm(w[i], 0x4b000000u, 0x7653)) - 8388736.f) * scale;
  }
}

__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {      // of bf16 pairs, NaN where either is
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The block of this thread's group of eight lanes: 8 values each, `left` of them inside the row.
template <bool VEC>
__device__ __forceinline__ void keep8(uint4 raw, int left, int8_t* q, float* scale, bool first) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  uint32_t top = max2_nan(max2_nan(raw.x & kAbs, raw.y & kAbs), max2_nan(raw.z & kAbs, raw.w & kAbs));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = max2_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  top = max2_nan(top, top >> 16);
  const ActScale k = act_scale(__uint_as_float(top << 16));
  if (first) *scale = k.scale;
  float v[8];
  spread(raw, v);
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = act_word(v[i], k.inv);      // (of a block that is not finite anything: its scale is NaN)
  const uint2 u = make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410),
                             __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410));
  if (VEC) {
    if (left > 0) *reinterpret_cast<uint2*>(q) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) q[i] = static_cast<int8_t>((i < 4 ? u.x : u.y) >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

constexpr int kGroups = kThreads / 8;      // blocks that a CTA works on at once

// A unit is a block of 64 columns of one row; a CTA takes UNROLL x kGroups neighbours at a time, each thread group every kGroups-th.
// Where a unit lies: row, first column of this lane, columns from there to the end of the row (0 or less: nothing).
struct Unit {
  int64_t row;
  int b, c, left;
  __device__ __forceinline__ Unit(uint32_t u, uint32_t units, const FastDiv& per_row, int width) {
    const bool in = u < units;
    const uint32_t r = in ? per_row(u) : 0u;
    row = r;
    b = in ? static_cast<int>(u - r * per_row.d) : 0;
    c = b * kActBlock + (threadIdx.x & 7) * 8;
    left = in ? width - c : 0;
  }
};

template <bool VEC>
__global__ void __launch_bounds__(kThreads, 5)
quantize8_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, float* __restrict__ scales, uint32_t units, int N,
                 FastDiv nb) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int U = 4;
  for (uint32_t u0 = blockIdx.x * (U * kGroups) + (threadIdx.x >> 3); u0 - (threadIdx.x >> 3) < units; u0 += gridDim.x * (U * kGroups)) {
    uint4 v[U];
    int64_t to[U];
    int left[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const Unit at(u0 + i * kGroups, units, nb, N);
      v[i] = load_raw<VEC>(x + at.row * ldx + at.c, at.left);
      to[i] = at.row * N + at.c;
      left[i] = at.left;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t u = u0 + i * kGroups;
      keep8<VEC>(v[i], left[i], q + to[i], scales + u, u < units && (threadIdx.x & 7) == 0);
    }
  }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads)
dequantize8_kernel(const int8_t* __restrict__ q, const float* __restrict__ scales, __nv_bfloat16* __restrict__ x, uint32_t units, int N,
                   FastDiv nb) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int U = 4;
  for (uint32_t u0 = blockIdx.x * (U * kGroups) + (threadIdx.x >> 3); u0 < units; u0 += gridDim.x * (U * kGroups)) {
    uint2 raw[U];
    float scale[U];
    int64_t to[U];
    int left[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t u = u0 + i * kGroups;
      const Unit at(u, units, nb, N);
      to[i] = at.row * N + at.c;
      left[i] = at.left;
      raw[i] = load_q<VEC>(q + to[i], at.left);
      scale[i] = u < units ? scales[u] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float v[8];
      read_q(raw[i], scale[i], v);
      store8<VEC>(x + to[i], left[i], v);
    }
  }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads, 4)
swiglu8_fwd_kernel(const __nv_bfloat16* __restrict__ gu, int64_t ldgu, __nv_bfloat16* __restrict__ act, int8_t* __restrict__ q,
                   float* __restrict__ scales, uint32_t units, int F, FastDiv nb) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int U = 2;
  for (uint32_t u0 = blockIdx.x * (U * kGroups) + (threadIdx.x >> 3); u0 - (threadIdx.x >> 3) < units; u0 += gridDim.x * (U * kGroups)) {
    uint4 gate[U], up[U];
    int64_t row[U];
    int c[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const Unit at(u0 + i * kGroups, units, nb, F);
      gate[i] = load_raw<VEC>(gu + at.row * ldgu + at.c, at.left);
      up[i] = load_raw<VEC>(gu + at.row * ldgu + F + at.c, at.left);
      row[i] = at.row;
      c[i] = at.left > 0 ? at.c : F;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t u = u0 + i * kGroups;
      const int left = F - c[i];
      float g[8], v[8], out[8];
      spread(gate[i], g);
      spread(up[i], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = g[j] * sigmoid(g[j]) * v[j];
      const int64_t at = row[i] * F + c[i];
      store8<VEC>(act + at, left, out);
      const bool first = u < units && (threadIdx.x & 7) == 0;
      float* scale = scales + (u + row[i] * static_cast<int>(nb.d));
      int8_t* to = q + (at + row[i] * F);
      keep8<VEC>(gate[i], left, to, scale, first);
      keep8<VEC>(up[i], left, to + F, scale + nb.d, first);
    }
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
__global__ void __launch_bounds__(kThreads, 4)
swiglu8_bwd_kernel(const __nv_bfloat16* __restrict__ dact, int64_t ldd, const int8_t* __restrict__ q, const float* __restrict__ scales,
                   __nv_bfloat16* __restrict__ dgu, uint32_t units, int F, FastDiv nb) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int U = 2;
  for (uint32_t u0 = blockIdx.x * (U * kGroups) + (threadIdx.x >> 3); u0 < units; u0 += gridDim.x * (U * kGroups)) {
    uint2 gate[U], up[U];
    uint4 d[U];
    float sg[U], su[U];
    int64_t to[U];
    int left[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t u = u0 + i * kGroups;
      const Unit at(u, units, nb, F);
      const float* scale = scales + (u + at.row * static_cast<int>(nb.d));
      to[i] = at.row * 2 * F + at.c;
      left[i] = at.left;
      gate[i] = load_q<VEC>(q + to[i], at.left);
      up[i] = load_q<VEC>(q + to[i] + F, at.left);
      sg[i] = u < units ? scale[0] : 0.f;
      su[i] = u < units ? scale[nb.d] : 0.f;
      d[i] = load_raw<VEC>(dact + at.row * ldd + at.c, at.left);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float g[8], u[8], da[8], dg[8], du[8];
      read_q(gate[i], sg[i], g);
      read_q(up[i], su[i], u);
      spread(d[i], da);
      swiglu_grad(g, u, da, dg, du);
      store8<VEC>(dgu + to[i], left[i], dg);
      store8<VEC>(dgu + to[i] + F, left[i], du);
    }
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
#pragma unroll 2
      for (int c = lane * 8; c < F; c += 256) {
        const int left = F - c;
        float gate[8], up[8], d[8], dg[8], du[8], a[8];
        if (Q8) {
          read_q(load_q<VEC>(q + row * 2 * F + c, left), scales[row * 2 * nb + c / kActBlock], gate);
          read_q(load_q<VEC>(q + row * 2 * F + F + c, left), scales[row * 2 * nb + nb + c / kActBlock], up);
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
  const dim3 grid(grid_for(M * nb, 4 * kGroups)), block(kThreads);
  const uint32_t units = static_cast<uint32_t>(M * nb);
  if (N % 8 == 0 && ldx % 8 == 0 && at16(x) && at16(q)) launch_pdl(quantize8_kernel<true>, grid, block, 0, stream, x, ldx, q, scales, units, N, FastDiv(nb));
  else launch_pdl(quantize8_kernel<false>, grid, block, 0, stream, x, ldx, q, scales, units, N, FastDiv(nb));
}

void dequantize8(const int8_t* q, const float* scales, __nv_bfloat16* x, int64_t M, int N, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return;
  const int nb = blocks_of(N);
  const dim3 grid(grid_for(M * nb, 4 * kGroups)), block(kThreads);
  const uint32_t units = static_cast<uint32_t>(M * nb);
  if (N % 8 == 0 && at16(x) && at16(q)) launch_pdl(dequantize8_kernel<true>, grid, block, 0, stream, q, scales, x, units, N, FastDiv(nb));
  else launch_pdl(dequantize8_kernel<false>, grid, block, 0, stream, q, scales, x, units, N, FastDiv(nb));
}

void swiglu8_fwd(const __nv_bfloat16* gu, int64_t ldgu, __nv_bfloat16* act, int8_t* q, float* scales, int64_t M, int F,
                 cudaStream_t stream) {
  if (M <= 0 || F <= 0) return;
  const int nb = blocks_of(F);
  const dim3 grid(grid_for(M * nb, 2 * kGroups)), block(kThreads);
  const uint32_t units = static_cast<uint32_t>(M * nb);
  if (F % 8 == 0 && ldgu % 8 == 0 && at16(gu) && at16(act) && at16(q))
    launch_pdl(swiglu8_fwd_kernel<true>, grid, block, 0, stream, gu, ldgu, act, q, scales, units, F, FastDiv(nb));
  else launch_pdl(swiglu8_fwd_kernel<false>, grid, block, 0, stream, gu, ldgu, act, q, scales, units, F, FastDiv(nb));
}

void swiglu8_bwd(const __nv_bfloat16* dact, int64_t ldd, const int8_t* q, const float* scales, __nv_bfloat16* dgu, int64_t M, int F,
                 cudaStream_t stream) {
  if (M <= 0 || F <= 0) return;
  const int nb = blocks_of(F);
  const dim3 grid(grid_for(M * nb, 2 * kGroups)), block(kThreads);
  const uint32_t units = static_cast<uint32_t>(M * nb);
  if (F % 8 == 0 && ldd % 8 == 0 && at16(dact) && at16(dgu) && at16(q))
    launch_pdl(swiglu8_bwd_kernel<true>, grid, block, 0, stream, dact, ldd, q, scales, dgu, units, F, FastDiv(nb));
  else launch_pdl(swiglu8_bwd_kernel<false>, grid, block, 0, stream, dact, ldd, q, scales, dgu, units, F, FastDiv(nb));
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
