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
// 32 to read back, and SwiGLU of 16384 x 1536 54 and 42; now 22, 18, 34 and 33 (128 and 204 MB).  Without gradients SwiGLU writes no
// checkpoint: 24 (151 MB).
//
// Widths that are no multiple of 8: a CTA takes whole rows, which lie one behind the other, brings them into shared memory as they lie (16
// bytes at a time, the ends value by value), works on them there and sends its results out the same way: 16384 x 2557 in 55 us to quantise
// and 42 to read back (value by value from memory 71 and 118), SwiGLU of 16384 x 1533 in 90 forward and 91 backward.  What bounds it are the
// 2-byte accesses to shared memory; rows shifted onto 16 bytes there instead, so that eight values go at once, took 68 and 56, 139 and 144:
// each 16 bytes are then read twice.  Rows that do not follow one another, or do not fit, go value by value from memory.
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

__device__ __forceinline__ float max_nan(float a, float b) {      // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
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

// KEEP: gate and up are written in 8 bits beside the activation (without gradients nobody reads them)
template <bool VEC, bool KEEP>
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
      if constexpr (!KEEP) continue;
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

// ---- rows of any width, through shared memory --------------------------------------------------------
// `bytes` from global memory to shared memory, `to` with the source's remainder by 16 (stage_at); by all threads of the CTA.
__device__ __forceinline__ uint8_t* stage_at(uint8_t* area, const void* p) { return area + (reinterpret_cast<uintptr_t>(p) & 15); }
__device__ __forceinline__ void stage_in(uint8_t* to, const void* from, int bytes) {
  const uint8_t* src = static_cast<const uint8_t*>(from);
  const int head = min(bytes, static_cast<int>(-reinterpret_cast<uintptr_t>(from) & 15)), body = (bytes - head) / 16;
  for (int i = threadIdx.x; i < head; i += kThreads) to[i] = src[i];
#pragma unroll 4
  for (int i = threadIdx.x; i < body; i += kThreads)
    *reinterpret_cast<uint4*>(to + head + i * 16) = *reinterpret_cast<const uint4*>(src + head + i * 16);
  for (int i = head + body * 16 + threadIdx.x; i < bytes; i += kThreads) to[i] = src[i];
}
__device__ __forceinline__ void stage_out(void* to, const uint8_t* from, int bytes) {
  uint8_t* dst = static_cast<uint8_t*>(to);
  const int head = min(bytes, static_cast<int>(-reinterpret_cast<uintptr_t>(to) & 15)), body = (bytes - head) / 16;
  for (int i = threadIdx.x; i < head; i += kThreads) dst[i] = from[i];
#pragma unroll 4
  for (int i = threadIdx.x; i < body; i += kThreads)
    *reinterpret_cast<uint4*>(dst + head + i * 16) = *reinterpret_cast<const uint4*>(from + head + i * 16);
  for (int i = head + body * 16 + threadIdx.x; i < bytes; i += kThreads) dst[i] = from[i];
}
// Value i of this lane's eight of a block: eight apart, so that eight lanes read neighbours, and turned by the warp's other blocks, which
// lie 128 bytes (64 as bytes) further on.
__device__ __forceinline__ int odd_place(int i) { return ((i + 2 * ((threadIdx.x >> 3) & 3)) & 7) * 8 + (threadIdx.x & 7); }
__device__ __forceinline__ float odd_load(const uint8_t* row, int c, int width) {
  return c < width ? __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[c]) << 16) : 0.f;
}
__device__ __forceinline__ void odd_store(uint8_t* row, int c, int width, float v) {
  if (c < width) reinterpret_cast<__nv_bfloat16*>(row)[c] = __float2bfloat16(v);
}
// keep8 for a block in shared memory
__device__ __forceinline__ void odd_keep(const float (&v)[8], uint8_t* q, int c0, int width, float* scale, bool in) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max_nan(a, fabsf(v[i]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  const ActScale k = act_scale(a);
  if (in && (threadIdx.x & 7) == 0) *scale = k.scale;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = c0 + odd_place(i);
    if (in && c < width) q[c] = act_byte(v[i], k.inv);
  }
}
// What a staged byte stands for
__device__ __forceinline__ float odd_read(const uint8_t* q, int c, int width, float scale) {
  return c < width ? static_cast<float>(static_cast<int8_t>(q[c])) * scale : 0.f;
}

constexpr int kOddValues = 8192;      // values of the widest tensor of a tile; wider rows are read from memory

// rows: of a tile.  Shared memory: the areas of what comes in and goes out, 16 bytes longer than they are and on 16 bytes.
__global__ void __launch_bounds__(kThreads)
quantize8_rows_kernel(const __nv_bfloat16* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scales, int64_t M, int N, int nb,
                      int rows) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ __align__(16) uint8_t area[];
  const int x_area = (rows * N * 2 + 31) / 16 * 16;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * rows; r0 < M; r0 += static_cast<int64_t>(gridDim.x) * rows) {
    const int n = static_cast<int>(M - r0 < rows ? M - r0 : rows);
    uint8_t* sx = stage_at(area, x + r0 * N);
    uint8_t* sq = stage_at(area + x_area, q + r0 * N);
    stage_in(sx, x + r0 * N, n * N * 2);
    __syncthreads();
    for (int u0 = threadIdx.x >> 5 << 2; u0 < n * nb; u0 += kGroups) {      // whole warps: four blocks
      const int u = u0 + ((threadIdx.x & 31) >> 3), row = u / nb, c0 = (u - row * nb) * kActBlock;
      const bool in = u < n * nb;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = in ? odd_load(sx + row * N * 2, c0 + odd_place(i), N) : 0.f;
      odd_keep(v, sq + row * N, c0, N, scales + r0 * nb + u, in);
    }
    __syncthreads();
    stage_out(q + r0 * N, sq, n * N);
  }
}

__global__ void __launch_bounds__(kThreads)
dequantize8_rows_kernel(const int8_t* __restrict__ q, const float* __restrict__ scales, __nv_bfloat16* __restrict__ x, int64_t M, int N, int nb,
                        int rows) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ __align__(16) uint8_t area[];
  const int x_area = (rows * N * 2 + 31) / 16 * 16;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * rows; r0 < M; r0 += static_cast<int64_t>(gridDim.x) * rows) {
    const int n = static_cast<int>(M - r0 < rows ? M - r0 : rows);
    uint8_t* sx = stage_at(area, x + r0 * N);
    uint8_t* sq = stage_at(area + x_area, q + r0 * N);
    stage_in(sq, q + r0 * N, n * N);
    __syncthreads();
    for (int u = threadIdx.x >> 3; u < n * nb; u += kGroups) {
      const int row = u / nb, c0 = (u - row * nb) * kActBlock;
      const float scale = scales[r0 * nb + u];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + odd_place(i);
        odd_store(sx + row * N * 2, c, N, odd_read(sq + row * N, c, N, scale));
      }
    }
    __syncthreads();
    stage_out(x + r0 * N, sx, n * N * 2);
  }
}

template <bool KEEP>
__global__ void __launch_bounds__(kThreads)
swiglu8_fwd_rows_kernel(const __nv_bfloat16* __restrict__ gu, __nv_bfloat16* __restrict__ act, int8_t* __restrict__ q,
                        float* __restrict__ scales, int64_t M, int F, int nb, int rows) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ __align__(16) uint8_t area[];
  const int gu_area = (rows * F * 4 + 31) / 16 * 16, act_area = (rows * F * 2 + 31) / 16 * 16;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * rows; r0 < M; r0 += static_cast<int64_t>(gridDim.x) * rows) {
    const int n = static_cast<int>(M - r0 < rows ? M - r0 : rows);
    uint8_t* sg = stage_at(area, gu + r0 * 2 * F);
    uint8_t* sa = stage_at(area + gu_area, act + r0 * F);
    uint8_t* sq = stage_at(area + gu_area + act_area, q + r0 * 2 * F);
    stage_in(sg, gu + r0 * 2 * F, n * F * 4);
    __syncthreads();
    for (int u0 = threadIdx.x >> 5 << 2; u0 < n * nb; u0 += kGroups) {
      const int u = u0 + ((threadIdx.x & 31) >> 3), row = u / nb, b = u - row * nb, c0 = b * kActBlock;
      const bool in = u < n * nb;
      float gate[8], up[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + odd_place(i);
        gate[i] = in ? odd_load(sg + row * F * 4, c, F) : 0.f;
        up[i] = in ? odd_load(sg + row * F * 4 + F * 2, c, F) : 0.f;
        if (in) odd_store(sa + row * F * 2, c, F, gate[i] * sigmoid(gate[i]) * up[i]);
      }
      if constexpr (!KEEP) continue;
      float* scale = scales + (r0 + row) * 2 * nb + b;
      odd_keep(gate, sq + row * 2 * F, c0, F, scale, in);
      odd_keep(up, sq + row * 2 * F + F, c0, F, scale + nb, in);
    }
    __syncthreads();
    stage_out(act + r0 * F, sa, n * F * 2);
    if constexpr (KEEP) stage_out(q + r0 * 2 * F, sq, n * F * 2);
  }
}

__global__ void __launch_bounds__(kThreads)
swiglu8_bwd_rows_kernel(const __nv_bfloat16* __restrict__ dact, const int8_t* __restrict__ q, const float* __restrict__ scales,
                        __nv_bfloat16* __restrict__ dgu, int64_t M, int F, int nb, int rows) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ __align__(16) uint8_t area[];
  const int gu_area = (rows * F * 4 + 31) / 16 * 16, act_area = (rows * F * 2 + 31) / 16 * 16;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * rows; r0 < M; r0 += static_cast<int64_t>(gridDim.x) * rows) {
    const int n = static_cast<int>(M - r0 < rows ? M - r0 : rows);
    uint8_t* sg = stage_at(area, dgu + r0 * 2 * F);
    uint8_t* sa = stage_at(area + gu_area, dact + r0 * F);
    uint8_t* sq = stage_at(area + gu_area + act_area, q + r0 * 2 * F);
    stage_in(sa, dact + r0 * F, n * F * 2);
    stage_in(sq, q + r0 * 2 * F, n * F * 2);
    __syncthreads();
    for (int u = threadIdx.x >> 3; u < n * nb; u += kGroups) {
      const int row = u / nb, b = u - row * nb, c0 = b * kActBlock;
      const float* scale = scales + (r0 + row) * 2 * nb + b;
      const float sgate = scale[0], sup = scale[nb];
      float g[8], v[8], d[8], dg[8], du[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + odd_place(i);
        g[i] = odd_read(sq + row * 2 * F, c, F, sgate);
        v[i] = odd_read(sq + row * 2 * F + F, c, F, sup);
        d[i] = odd_load(sa + row * F * 2, c, F);
      }
      swiglu_grad(g, v, d, dg, du);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + odd_place(i);
        odd_store(sg + row * F * 4, c, F, dg[i]);
        odd_store(sg + row * F * 4 + F * 2, c, F, du[i]);
      }
    }
    __syncthreads();
    stage_out(dgu + r0 * 2 * F, sg, n * F * 4);
  }
}

// One warp per choice: the row of its gradient and the dot product that is its weight's.  s comes in bf16, and d(gate), d(up) and the weighted
// activation leave in bf16: they are operands of the next products; what is done with them here is fp32.  Bound by memory: 16384 x 1536 in
// 51 us (302 MB, 5.9 TB/s).
template <bool Q8>
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
          read_q(load_q<true>(q + row * 2 * F + c, left), scales[row * 2 * nb + c / kActBlock], gate);
          read_q(load_q<true>(q + row * 2 * F + F + c, left), scales[row * 2 * nb + nb + c / kActBlock], up);
        } else {
          load8<true>(gu + row * 2 * F + c, left, gate);
          load8<true>(gu + row * 2 * F + F + c, left, up);
        }
        load8<true>(s + row * F + c, left, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a[j] = gate[j] * sigmoid(gate[j]) * up[j];
          dot = fmaf(a[j], d[j], dot);
          a[j] *= w;
          d[j] *= w;
        }
        swiglu_grad(gate, up, d, dg, du);
        store8<true>(act_w + row * F + c, left, a);
        store8<true>(dgu + row * 2 * F + c, left, dg);
        store8<true>(dgu + row * 2 * F + F + c, left, du);
      }
      dot = warp_sum(dot);
    }
    if (lane == 0) dweights[i] = dot;
    if (i >= live) {      // row i is no choice's
      const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int c = lane * 8; c < F; c += 256) {
        store8<true>(act_w + static_cast<int64_t>(i) * F + c, F - c, zero);
        store8<true>(dgu + static_cast<int64_t>(i) * 2 * F + c, F - c, zero);
        store8<true>(dgu + static_cast<int64_t>(i) * 2 * F + F + c, F - c, zero);
      }
    }
  }
}

int blocks_of(int n) { return (n + kActBlock - 1) / kActBlock; }
int grid_for(int64_t units, int per_cta) {
  const int64_t need = (units + per_cta - 1) / per_cta;
  return static_cast<int>(need < 148 * 16 ? need : 148 * 16);
}
// Rows of a tile that go through shared memory; `width`: of the widest tensor
int tile_rows(int64_t M, int width) {
  const int fit = kOddValues / width;
  const int64_t spread = (M + 148 * 6 - 1) / (148 * 6);      // small matrices: over all SMs
  return static_cast<int>(spread < 1 ? 1 : spread < fit ? spread : fit);
}
int tile_grid(int64_t M, int rows) {
  const int64_t need = (M + rows - 1) / rows;
  return static_cast<int>(need < 148 * 8 ? need : 148 * 8);
}
bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int quantize8(const __nv_bfloat16* x, int64_t ldx, int8_t* q, float* scales, int64_t M, int N, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  const int nb = blocks_of(N);
  const dim3 grid(grid_for(M * nb, 4 * kGroups)), block(kThreads);
  const uint32_t units = static_cast<uint32_t>(M * nb);
  cudaError_t rc;
  if (N % 8 == 0 && ldx % 8 == 0 && at16(x) && at16(q)) {
    rc = launch_pdl(quantize8_kernel<true>, grid, block, 0, stream, x, ldx, q, scales, units, N, FastDiv(nb));
  } else if (ldx == N && N <= kOddValues) {
    const int rows = tile_rows(M, N);
    rc = launch_pdl(quantize8_rows_kernel, dim3(tile_grid(M, rows)), block, rows * N * 3 + 64, stream, x, q, scales, M, N, nb, rows);
  } else {
    rc = launch_pdl(quantize8_kernel<false>, grid, block, 0, stream, x, ldx, q, scales, units, N, FastDiv(nb));
  }
  return launch_code(rc);
}

int dequantize8(const int8_t* q, const float* scales, __nv_bfloat16* x, int64_t M, int N, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  const int nb = blocks_of(N);
  const dim3 grid(grid_for(M * nb, 4 * kGroups)), block(kThreads);
  const uint32_t units = static_cast<uint32_t>(M * nb);
  cudaError_t rc;
  if (N % 8 == 0 && at16(x) && at16(q)) {
    rc = launch_pdl(dequantize8_kernel<true>, grid, block, 0, stream, q, scales, x, units, N, FastDiv(nb));
  } else if (N <= kOddValues) {
    const int rows = tile_rows(M, N);
    rc = launch_pdl(dequantize8_rows_kernel, dim3(tile_grid(M, rows)), block, rows * N * 3 + 64, stream, q, scales, x, M, N, nb, rows);
  } else {
    rc = launch_pdl(dequantize8_kernel<false>, grid, block, 0, stream, q, scales, x, units, N, FastDiv(nb));
  }
  return launch_code(rc);
}

int swiglu8_fwd(const __nv_bfloat16* gu, int64_t ldgu, __nv_bfloat16* act, int8_t* q, float* scales, int64_t M, int F,
                 cudaStream_t stream) {
  if (M <= 0 || F <= 0) return 0;
  const int nb = blocks_of(F);
  const dim3 grid(grid_for(M * nb, 2 * kGroups)), block(kThreads);
  const uint32_t units = static_cast<uint32_t>(M * nb);
  cudaError_t rc;
  if (F % 8 == 0 && ldgu % 8 == 0 && at16(gu) && at16(act) && at16(q)) {
    rc = launch_pdl(q ? swiglu8_fwd_kernel<true, true> : swiglu8_fwd_kernel<true, false>, grid, block, 0, stream, gu, ldgu, act, q, scales, units,
                    F, FastDiv(nb));
  } else if (ldgu == 2 * static_cast<int64_t>(F) && 2 * F <= kOddValues) {
    const int rows = tile_rows(M, 2 * F);
    rc = launch_pdl(q ? swiglu8_fwd_rows_kernel<true> : swiglu8_fwd_rows_kernel<false>, dim3(tile_grid(M, rows)), block, rows * F * 8 + 96, stream,
                    gu, act, q, scales, M, F, nb, rows);
  } else {
    rc = launch_pdl(q ? swiglu8_fwd_kernel<false, true> : swiglu8_fwd_kernel<false, false>, grid, block, 0, stream, gu, ldgu, act, q, scales, units,
                    F, FastDiv(nb));
  }
  return launch_code(rc);
}

int swiglu8_bwd(const __nv_bfloat16* dact, int64_t ldd, const int8_t* q, const float* scales, __nv_bfloat16* dgu, int64_t M, int F,
                 cudaStream_t stream) {
  if (M <= 0 || F <= 0) return 0;
  const int nb = blocks_of(F);
  const dim3 grid(grid_for(M * nb, 2 * kGroups)), block(kThreads);
  const uint32_t units = static_cast<uint32_t>(M * nb);
  cudaError_t rc;
  if (F % 8 == 0 && ldd % 8 == 0 && at16(dact) && at16(dgu) && at16(q)) {
    rc = launch_pdl(swiglu8_bwd_kernel<true>, grid, block, 0, stream, dact, ldd, q, scales, dgu, units, F, FastDiv(nb));
  } else if (ldd == F && 2 * F <= kOddValues) {
    const int rows = tile_rows(M, 2 * F);
    rc = launch_pdl(swiglu8_bwd_rows_kernel, dim3(tile_grid(M, rows)), block, rows * F * 8 + 96, stream, dact, q, scales, dgu, M, F, nb, rows);
  } else {
    rc = launch_pdl(swiglu8_bwd_kernel<false>, grid, block, 0, stream, dact, ldd, q, scales, dgu, units, F, FastDiv(nb));
  }
  return launch_code(rc);
}

int expert_swiglu_bwd(const __nv_bfloat16* s, const __nv_bfloat16* gu, const int8_t* q, const float* scales, const float* weights,
                       const int* slots, const int* offsets, __nv_bfloat16* dgu, __nv_bfloat16* act_w, float* dweights, int R, int E,
                       int F, cudaStream_t stream) {
  if (R <= 0 || F <= 0) return 0;
  const int nb = blocks_of(F);
  const dim3 grid(grid_for(R, kWarps)), block(kThreads);
  return launch_code(launch_pdl(gu ? expert_swiglu_bwd_kernel<false> : expert_swiglu_bwd_kernel<true>, grid, block, 0, stream, s, gu, q, scales,
                                weights, slots, offsets, dgu, act_w, dweights, R, E, F, nb));
}

}  // namespace tb
