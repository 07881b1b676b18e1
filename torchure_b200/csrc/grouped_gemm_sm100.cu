// Matrix products of rows grouped by expert, each group with its expert's matrix, and the gradient of the matrices.
//
// One CTA per 64 x 64 tile of one expert's output, operands staged in shared memory as fp32, 4 x 4 sums per thread.  Bound by the
// FMA units: 32768 x 1024 x 1536 x 6 operations take 14.2 ms over 32 experts.
#include "common.cuh"
#include "moe_api.h"

namespace tb {

namespace {

constexpr int TILE = 64, KB = 16;

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// acc[i][j] += sum over k0 <= k < k1 of A(m0 + 4 ty + i, k) B(n0 + 4 tx + j, k), with A(m, k) = a[m * am + k * ak], zero from M / N on
__device__ __forceinline__ void tile_product(const __nv_bfloat16* a, int64_t am, int64_t ak, int m0, int M, const __nv_bfloat16* b,
                                             int64_t bm, int64_t bk, int n0, int N, int64_t k0, int64_t k1, float (&acc)[4][4]) {
  __shared__ float sa[KB][TILE + 1], sb[KB][TILE + 1];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  for (int64_t k = k0; k < k1; k += KB) {
    for (int i = tid; i < TILE * KB; i += 256) {
      // the faster index runs along the contiguous direction
      const int ka = ak == 1 ? i % KB : i / TILE, ma = ak == 1 ? i / KB : i % TILE;
      sa[ka][ma] = m0 + ma < M && k + ka < k1 ? __bfloat162float(a[(m0 + ma) * am + (k + ka) * ak]) : 0.f;
      const int kb = bk == 1 ? i % KB : i / TILE, mb = bk == 1 ? i / KB : i % TILE;
      sb[kb][mb] = n0 + mb < N && k + kb < k1 ? __bfloat162float(b[(n0 + mb) * bm + (k + kb) * bk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < KB; ++kk) {
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[i] = sa[kk][4 * ty + i]; y[i] = sb[kk][4 * tx + i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(256)
grouped_simple_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ w, int64_t wn, int64_t wk,
                      const int* __restrict__ offsets, __nv_bfloat16* __restrict__ y, int R, int E, int N, int K) {
  // tile blockIdx.y of the row tiles of all groups, the rows of no expert being the last group
  int left = blockIdx.y, lo = 0, hi = 0, e = 0;
  for (; e <= E; ++e) {
    lo = hi;
    hi = e < E ? min(max(offsets[e + 1], lo), R) : R;
    const int tiles = (hi - lo + TILE - 1) / TILE;
    if (left < tiles) break;
    left -= tiles;
  }
  if (e > E) return;
  const int m0 = lo + left * TILE, n0 = blockIdx.x * TILE;
  float acc[4][4] = {};
  if (e < E)
    tile_product(x, ldx, 1, m0, hi, w + static_cast<int64_t>(e) * N * K, wn, wk, n0, N, 0, K, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + 4 * ty + i, n = n0 + 4 * tx + j;
      if (m < hi && n < N) y[static_cast<int64_t>(m) * N + n] = __float2bfloat16(acc[i][j]);
    }
}

template <class O>
__global__ void __launch_bounds__(256)
grouped_wgrad_simple_kernel(const __nv_bfloat16* __restrict__ dy, int64_t lddy, const __nv_bfloat16* __restrict__ x, int64_t ldx,
                            const int* __restrict__ offsets, O* __restrict__ dw, int R, int N, int K) {
  const int e = blockIdx.z;
  int lo = 0;
  for (int i = 1; i <= e; ++i) lo = min(max(offsets[i], lo), R);
  const int hi = min(max(offsets[e + 1], lo), R);
  const int n0 = blockIdx.y * TILE, k0 = blockIdx.x * TILE;
  float acc[4][4] = {};
  tile_product(dy, 1, lddy, n0, N, x, 1, ldx, k0, K, lo, hi, acc);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 4 * ty + i, k = k0 + 4 * tx + j;
      if (n < N && k < K) put(dw + (static_cast<int64_t>(e) * N + n) * K + k, acc[i][j]);
    }
}

}  // namespace

int grouped_gemm(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* w, bool w_t, const int* offsets, __nv_bfloat16* y, int R,
                 int E, int N, int K, int* err, int num_sms, cudaStream_t stream) {
  const dim3 grid((N + TILE - 1) / TILE, (R + TILE - 1) / TILE + E + 1);
  if (grid.y > 65535) return -3;
  grouped_simple_kernel<<<grid, 256, 0, stream>>>(x, ldx, w, w_t ? 1 : K, w_t ? N : 1, offsets, y, R, E, N, K);
  return cudaGetLastError() == cudaSuccess ? 0 : -21;
}

int grouped_wgrad(const __nv_bfloat16* dy, int64_t lddy, const __nv_bfloat16* x, int64_t ldx, const int* offsets, void* dw, bool dw_bf16,
                  int R, int E, int N, int K, int* err, int num_sms, cudaStream_t stream) {
  const dim3 grid((K + TILE - 1) / TILE, (N + TILE - 1) / TILE, E);
  if (dw_bf16)
    grouped_wgrad_simple_kernel<<<grid, 256, 0, stream>>>(dy, lddy, x, ldx, offsets, static_cast<__nv_bfloat16*>(dw), R, N, K);
  else
    grouped_wgrad_simple_kernel<<<grid, 256, 0, stream>>>(dy, lddy, x, ldx, offsets, static_cast<float*>(dw), R, N, K);
  return cudaGetLastError() == cudaSuccess ? 0 : -21;
}

}  // namespace tb
