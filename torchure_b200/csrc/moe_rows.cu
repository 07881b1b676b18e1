// Rows between token order and expert order: gather (dispatch), weighted sum (combine), and the gradient of the sum.
//
// All three move each byte once and are bound by memory; 8 columns per lane, 16-byte accesses of bf16 rows.  The gather gives a row to a
// warp, with four loads on their way per lane (8192 x 1024 to 16384 rows 9.5 us, 15 with one).  The sum gives 8 columns of a token to a
// thread and keeps an SM full of threads, four choices' loads on their way each: one warp per token with as many loads took 19.5 us
// for the same rows, short-lived warps that each wait for slots, then for rows; now 12.4.  The gradient of the sum gives a choice to a warp
// (13.5 for the same).  Rows that are no multiple of 8 columns or start
// off a 16-byte boundary are read value by value.
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

// 8 values as they lie in memory, `left` of them inside the row, zeros behind
template <class T>
struct Packed;
template <>
struct Packed<__nv_bfloat16> {
  uint4 raw;
  template <bool VEC>
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int left) {
    if (VEC) {
      raw = left > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
      return;
    }
    uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) u[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
    raw = make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ __forceinline__ void add(float w, float (&sum)[8]) const {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      sum[2 * n] = fmaf(w, __uint_as_float(u[n] << 16), sum[2 * n]);
      sum[2 * n + 1] = fmaf(w, __uint_as_float(u[n] & 0xffff0000u), sum[2 * n + 1]);
    }
  }
};
template <>
struct Packed<float> {
  float v[8];
  template <bool VEC>
  __device__ __forceinline__ void load(const float* p, int left) {
    if (VEC && left > 0) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
  }
  __device__ __forceinline__ void add(float w, float (&sum)[8]) const {
#pragma unroll
    for (int n = 0; n < 8; ++n) sum[n] = fmaf(w, v[n], sum[n]);
  }
};

// 8 values from column c of a row of D
template <bool VEC>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int c, int D, float (&v)[8]) {
  if (VEC) {
    const uint4 u = *reinterpret_cast<const uint4*>(p + c);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < D ? __bfloat162float(p[c + i]) : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int c, int D, float (&v)[8]) {
  if (VEC) {
    const float4 a = *reinterpret_cast<const float4*>(p + c), b = *reinterpret_cast<const float4*>(p + c + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < D ? p[c + i] : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(__nv_bfloat16* p, int c, int D, const float (&v)[8]) {
  if (VEC) {
    *reinterpret_cast<uint4*>(p + c) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < D) p[c + i] = __float2bfloat16(v[i]);
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(float* p, int c, int D, const float (&v)[8]) {
  if (VEC) {
    *reinterpret_cast<float4*>(p + c) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < D) p[c + i] = v[i];
  }
}

template <class X, bool VEC>
__global__ void __launch_bounds__(kThreads)
rows_gather_kernel(const X* __restrict__ x, int64_t ldx, const int* __restrict__ rows, __nv_bfloat16* __restrict__ out, int T, int k,
                   int R, int D) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  for (int r = blockIdx.x * kWarps + (threadIdx.x >> 5); r < R; r += gridDim.x * kWarps) {
    const int i = rows[r];
    const int t = i < 0 ? -1 : i / k;
    const bool live = t >= 0 && t < T;
    const X* src = x + (live ? t : 0) * ldx;
    __nv_bfloat16* dst = out + static_cast<int64_t>(r) * D;
    for (int c0 = lane * 8; c0 < D; c0 += 1024) {
      float v[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
        if (live && c0 + u * 256 < D) load8<VEC>(src, c0 + u * 256, D, v[u]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c0 + u * 256 < D) store8<VEC>(dst, c0 + u * 256, D, v[u]);
    }
  }
}

// One thread per 8 columns of a token.  chunks: of 8 columns in a row.
template <class Y, class O, bool VEC>
__global__ void __launch_bounds__(kThreads)
rows_combine_kernel(const Y* __restrict__ y, const float* __restrict__ weights, const int* __restrict__ slots, O* __restrict__ out,
                    int64_t total, int k, int R, int D, FastDiv chunks) {
  pdl_wait();
  pdl_launch_dependents();
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const uint32_t t = chunks(static_cast<uint32_t>(i));
    const int c = static_cast<int>(static_cast<uint32_t>(i) - t * chunks.d) * 8;
    const int64_t i0 = static_cast<int64_t>(t) * k;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < k; j0 += 4) {
      Packed<Y> raw[4];
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j0 + j < k ? slots[i0 + j0 + j] : -1;
        const bool in = r >= 0 && r < R;
        w[j] = in ? (weights ? weights[i0 + j0 + j] : 1.f) : 0.f;
        raw[j].template load<VEC>(y + static_cast<int64_t>(in ? r : 0) * D + c, in ? D - c : 0);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j].add(w[j], sum);
    }
    store8<VEC>(out + static_cast<int64_t>(t) * D, c, D, sum);
  }
}

template <class O, bool VEC>
__global__ void __launch_bounds__(kThreads)
rows_combine_bwd_kernel(const O* __restrict__ dout, int64_t ld, const __nv_bfloat16* __restrict__ y,
                        const float* __restrict__ weights, const int* __restrict__ slots, const int* __restrict__ offsets,
                        __nv_bfloat16* __restrict__ dy, float* __restrict__ dweights, int T, int k, int E, int D) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int R = T * k;
  const int live = min(max(offsets[E], 0), R);
  for (int i = blockIdx.x * kWarps + (threadIdx.x >> 5); i < R; i += gridDim.x * kWarps) {
    const int r = slots[i];
    float dot = 0.f;
    if (r >= 0 && r < R) {
      const O* d = dout + (i / k) * ld;
      const float w = weights[i];
#pragma unroll 2
      for (int c = lane * 8; c < D; c += 256) {
        float a[8], b[8];
        load8<VEC>(d, c, D, a);
        load8<VEC>(y + static_cast<int64_t>(r) * D, c, D, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dot = fmaf(a[j], b[j], dot);
          a[j] *= w;
        }
        store8<VEC>(dy + static_cast<int64_t>(r) * D, c, D, a);
      }
      dot = warp_sum(dot);
    }
    if (lane == 0) dweights[i] = dot;
    if (i >= live) {      // row i is no choice's
      const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int c = lane * 8; c < D; c += 256) store8<VEC>(dy + static_cast<int64_t>(i) * D, c, D, zero);
    }
  }
}

int grid_for(int rows) {
  const int need = (rows + kWarps - 1) / kWarps;
  return need < 148 * 8 ? need : 148 * 8;
}

bool whole(const void* p, int64_t ld, int D) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && D % 8 == 0; }

}  // namespace

int rows_gather(const void* x, bool x_bf16, int64_t ldx, const int* rows, __nv_bfloat16* out, int T, int k, int R, int D,
                 cudaStream_t stream) {
  if (R <= 0 || D <= 0) return 0;
  const dim3 grid(grid_for(R)), block(kThreads);
  const bool vec = whole(x, ldx, D) && whole(out, D, D);
  cudaError_t rc;
#define TB_GATHER(X, V) rc = launch_pdl(rows_gather_kernel<X, V>, grid, block, 0, stream, static_cast<const X*>(x), ldx, rows, out, T, k, R, D)
  if (x_bf16) { if (vec) TB_GATHER(__nv_bfloat16, true); else TB_GATHER(__nv_bfloat16, false); }
  else { if (vec) TB_GATHER(float, true); else TB_GATHER(float, false); }
#undef TB_GATHER
  return launch_code(rc);
}

int rows_combine(const void* y, bool y_bf16, const float* weights, const int* slots, void* out, bool out_bf16, int T, int k, int R, int D,
                  cudaStream_t stream) {
  if (T <= 0 || D <= 0) return 0;
  const int chunks = (D + 7) / 8;
  const int64_t total = static_cast<int64_t>(T) * chunks, need = (total + kThreads - 1) / kThreads;
  const dim3 grid(static_cast<int>(need < 148 * 16 ? need : 148 * 16)), block(kThreads);
  const bool vec = whole(y, D, D) && whole(out, D, D);
  cudaError_t rc;
#define TB_COMBINE(Y, O, V)                                                                                                             \
  rc = launch_pdl(rows_combine_kernel<Y, O, V>, grid, block, 0, stream, static_cast<const Y*>(y), weights, slots, static_cast<O*>(out), \
                  total, k, R, D, FastDiv(chunks))
#define TB_COMBINE_OF(Y)                                                                                                 \
  if (out_bf16) { if (vec) TB_COMBINE(Y, __nv_bfloat16, true); else TB_COMBINE(Y, __nv_bfloat16, false); }               \
  else { if (vec) TB_COMBINE(Y, float, true); else TB_COMBINE(Y, float, false); }
  if (y_bf16) { TB_COMBINE_OF(__nv_bfloat16) } else { TB_COMBINE_OF(float) }
#undef TB_COMBINE_OF
#undef TB_COMBINE
  return launch_code(rc);
}

int rows_combine_bwd(const void* dout, bool dout_bf16, int64_t ld, const __nv_bfloat16* y, const float* weights, const int* slots,
                      const int* offsets, __nv_bfloat16* dy, float* dweights, int T, int k, int E, int D, cudaStream_t stream) {
  if (T <= 0 || D <= 0) return 0;
  const dim3 grid(grid_for(T * k)), block(kThreads);
  const bool vec = whole(dout, ld, D) && whole(y, D, D) && whole(dy, D, D);
  cudaError_t rc;
#define TB_COMBINE_BWD(O, V)                                                                                                              \
  rc = launch_pdl(rows_combine_bwd_kernel<O, V>, grid, block, 0, stream, static_cast<const O*>(dout), ld, y, weights, slots, offsets, dy, \
                  dweights, T, k, E, D)
  if (dout_bf16) { if (vec) TB_COMBINE_BWD(__nv_bfloat16, true); else TB_COMBINE_BWD(__nv_bfloat16, false); }
  else { if (vec) TB_COMBINE_BWD(float, true); else TB_COMBINE_BWD(float, false); }
#undef TB_COMBINE_BWD
  return launch_code(rc);
}

}  // namespace tb
