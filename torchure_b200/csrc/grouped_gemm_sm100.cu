// Matrix products of rows grouped by expert, each group with its expert's matrix, and the gradient of the matrices, on CTA pairs
// (tcgen05.mma.cta_group::2, 256 x 256 tiles over two SMs; the pipeline is that of gemm2_sm100.cu).
//
// Rows times matrices, y[r] = x[r] W[e(r)]^T: the tile is computed transposed.  The matrix supplies the 256 rows of the tile (the
// instruction's M, fixed), the group's rows its columns (the instruction's N, any multiple of 32 up to 256).  Groups end anywhere, and
// what a group's last tile costs in arithmetic goes with its rows: 2049 rows take 8.1 tiles, not 9.  Nothing is padded in memory: a
// tile reads rows of the next group along, whose columns of the tile are not stored.  The epilogue turns the accumulator round on its
// way out: fragments of 16 lanes x 8 columns (tcgen05.ld.16x256b) are rounded to pairs and stored transposed (stmatrix) into staging rows
// of four warps, from which the output leaves in whole lines of 128 bytes.
//
// The gradient of the matrices, dW[e] = sum of dy[r]^T x[r]: the group's rows are the reduction.  Blocks of 64 rows; of a last block
// that is not full only the steps of 16 rows that hold some are multiplied, and in a step that is not full the rows of the next group
// are overwritten with zeros in shared memory, in both operands (0 x NaN is NaN), by a warp that does nothing else.
//
// Groups are read from `offsets` on the device: no call waits for them.  The grid is persistent; tiles go round over the pairs.
//
// With SwiGLU in the epilogue the matrix is gate over up, and a CTA's 128 tile rows are four times 16 gate rows and the 16 up rows of
// the same units: a warp, which reads 32 lanes of the accumulator, has both factors of its 16 units, in the same place of two
// fragments.  The activation is taken from the fp32 sums; gate and up are stored beside it in bf16, or in 8 bits with a scale for the
// CTA's 64 units (act8.cu has the format), or not at all.
//
// Bound by the tensor cores at the clock that the power allows (1.58 GHz).  16384 rows in 8 uneven groups, 1024 x 2 x 1536: 74 us forward, 77
// for the rows' gradient, 76 for the matrices' (an equally large dense product 71), with SwiGLU 86 (73 if gate and up are not kept, 94 if in 8
// bits); 32768 rows in 32 groups, 1024 x 1536, back to back: 90, 89, 94.  All sums are fp32; results are rounded once, to bf16, which the next
// product reads (an output that is only added up, of few rows, stays fp32).
//
// Few rows per group: grouped_few_kernel, single CTAs on 128 tile rows and at most 64 group rows, two of them on an SM.  The matrices
// are then all the traffic there is, and what counts is how evenly it is spread and how many copies are on their way.  There the
// group's rows may be listed (places of token rows in expert order) and are gathered four to a copy (tile::gather4), which spares a
// launch.  A copy of four rows costs about 72 cycles, so that tiles of many rows do better with the rows put in order first (the pair
// kernels with listed rows took 270 us instead of 88 + 9.6).  In a feed-forward pass of few rows, whose launches overlap, the first tile of
// every group has a CTA that is known beforehand (EARLY): it asks for its first four blocks of the matrix while the kernel before is still at
// work.
#include "act8.cuh"
#include "cta_pair.cuh"
#include "moe_api.h"

namespace tb {

int make_tmap_2d(CUtensorMap* map, const void* base, int elem_bytes, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows,
                 uint32_t box_cols);
int make_tmap_3d(CUtensorMap* map, const void* base, int elem_bytes, uint64_t planes, uint64_t rows, uint64_t cols, uint32_t box_rows,
                 uint32_t box_cols);
int make_tmap_gate_up(CUtensorMap* map, const void* base, uint64_t planes, uint64_t rows, uint64_t cols, int groups);

namespace {

constexpr int BM = 128, BN = 256, BNH = 128, BK = 64, STAGES = 6;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BNH * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int BAR_BYTES = 240;
constexpr int EDGE_BYTES = (kMaxExperts + 1) * 4;
constexpr uint32_t TMEM_COLS = 512;

// Staged rows of the four epilogue warps that have a CTA's 128 accumulator lanes, 32 at a time, so that the output is written in whole
// lines of 128 bytes (in pieces of 32 bytes, a warp's own units, gate and up beside the activation took 103 us instead of 78 without
// them).  Eight rows of 272 or of 400 bytes fall on every bank once.
//   kStore    128 columns in bf16
//   kSwiglu   64 units: activation | gate | up in bf16
//   kSwiglu8  64 units: activation in bf16 | gate | up in 8 bits
//   kStore32  128 columns in fp32 (a few rows' products that are added up afterwards)
enum { kStore = 0, kSwiglu = 1, kSwiglu8 = 2, kStore32 = 3 };
template <int EPI>
constexpr bool kGateUp = EPI == kSwiglu || EPI == kSwiglu8;      // the matrix is gate over up
constexpr int EPI_ROWS = 32;
template <int EPI>
constexpr int kPitch = EPI == kStore32 ? 528 : EPI == kSwiglu ? 400 : 272;
// kSwiglu8, for the four warps: their largest magnitudes, and the reciprocals
constexpr int MAX_BYTES = 4 * 2 * EPI_ROWS * 2, INV_BYTES = 2 * EPI_ROWS * 4;
template <int EPI>
constexpr int kPartBytes = EPI_ROWS * kPitch<EPI> + (EPI == kSwiglu8 ? MAX_BYTES + INV_BYTES : 0);
constexpr int ROW_EPI_BYTES = 2 * kPartBytes<kSwiglu>;
static_assert(kPartBytes<kSwiglu8> <= kPartBytes<kSwiglu> && kPartBytes<kStore> <= kPartBytes<kSwiglu>, "staging rows");
constexpr int ROW_THREADS = 320;      // warp 0 copies, warp 1 issues the products, warps 2 - 9 are the epilogue
constexpr int FEW_THREADS = 192;
constexpr int ROW_SMEM = STAGES * STAGE_BYTES + ROW_EPI_BYTES + BAR_BYTES + EDGE_BYTES + 1024;

constexpr int EPI_BUF = 4096;                   // 32 rows x 128 B
constexpr int W_EPI_BYTES = 8 * EPI_BUF;        // a buffer for each of eight epilogue warps
constexpr int ORDERED = 256;                    // up to this many groups are taken in falling order of their rows
constexpr int W_THREADS = 352;                  // warp 0 copies, 1 issues the products, 2 - 9 are the epilogue, 10 zeroes rows
constexpr int W_SMEM = STAGES * STAGE_BYTES + W_EPI_BYTES + BAR_BYTES + EDGE_BYTES + ORDERED + 1024;
static_assert(ROW_SMEM <= 232448 && W_SMEM <= 232448, "shared memory of one CTA");

// edge[e] = first row of group e, edge[E] = end of the last: what `offsets` says, brought into [0, R] and made not to fall
__device__ __forceinline__ void load_edges(const int* offsets, int* edge, int E, int R) {
  if (threadIdx.x < 32) {
    int run = 0;
    for (int e0 = 0; e0 <= E; e0 += 32) {
      const int e = e0 + static_cast<int>(threadIdx.x);
      int v = e > 0 && e <= E ? min(max(offsets[e], 0), R) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, v, o);
        if (threadIdx.x >= o) v = max(v, up);
      }
      v = max(v, run);
      if (e <= E) edge[e] = v;
      run = __shfl_sync(0xffffffffu, v, 31);
    }
  }
}

// The units of group e are its tiles of 256 rows times `cols` tiles of the matrix, rows fastest; a pair takes every num_clusters-th.
// (With the units of the last, not full wave cut into pieces by rows, 3.46 waves as 3.6, nothing got faster: the clocks give what the
// idle SMs leave.)
struct Place {
  const int* edge;
  int E, cols;
  int e = 0, base = 0;      // base: first unit of group e
  // Where unit `unit` lies (it only grows from call to call): rows and column.  False: past the last.
  __device__ __forceinline__ bool find(int unit, int& r0, int& live, int& col) {
    while (e < E) {
      const int tiles = (edge[e + 1] - edge[e] + BN - 1) / BN;
      if (unit - base < tiles * cols) {
        const int at = unit - base;
        r0 = edge[e] + at % tiles * BN;
        live = min(BN, edge[e + 1] - r0);
        col = at / tiles;
        return true;
      }
      base += tiles * cols;
      ++e;
    }
    return false;
  }
};

// Where the rows of a product go.  width: columns of the output (units for SwiGLU); gu, q: one of them or neither
struct RowsOut {
  __nv_bfloat16* y;      // the product, or the activation; kStore32: nullptr
  __nv_bfloat16* gu;     // [R, 2 width]
  int8_t* q;             // [R, 2 width]
  float* scales;         // [R, 2 ceil(width / 64)]
  int width;
  float* y32;            // kStore32: the product
};

// Where the rows of x lie: row r is row list[r] / k of `count` rows; what the list calls none (-1) is row 0, whose results are not used.
struct Rows {
  const int* list;
  FastDiv k;
  int count;
  __device__ __forceinline__ int at(int r, int end) const {
    const int i = r < end ? list[r] : 0;
    return min(static_cast<int>(k(static_cast<uint32_t>(max(i, 0)))), count - 1);
  }
};

__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.f + __expf(-x)); }

__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {      // of bf16 pairs, NaN where either is
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The epilogue of four warps, of which this is number q4 with 32 accumulator lanes from t_row on: columns 0 .. live - 1 of the tile, which
// are rows r0 .. of the output; 32 of them at a time, from `from` on in steps of `step`.  n0: first output column (first unit) of the
// CTA's lanes; buf: kPartBytes of the four, bar: their named barrier.  release() once this warp has read the accumulator.
template <int EPI, class Release>
__device__ __forceinline__ void rows_epilogue(const RowsOut& out, uint32_t t_row, int q4, uint8_t* buf, int bar, int r0, int live, int from,
                                              int step, int n0, Release release) {
  const int lane = threadIdx.x & 31, tid = q4 * 32 + lane;
  const int N = out.width;
  constexpr int P = kPitch<EPI>;
  // stmatrix: this lane's row and tile
  const uint32_t put = smem_u32(buf) + (lane & 7) * P + q4 * (EPI == kStore ? 64 : 32) + (lane >> 3) * 16;
  if (from >= live) release();
#pragma unroll 1
  for (int c = from; c < live; c += step) {
    uint32_t v[16], u[16];
    __syncwarp();
    tmem_ld_16x256b_x4(t_row + c, v);
    tmem_ld_16x256b_x4(t_row + c + (16u << 16), u);
    tmem_ld_wait();
    if (c + step >= live) release();
    if constexpr (EPI == kStore32) {
      named_bar_sync(bar, 128);      // the rows staged before have been read
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int h = 0; h < 4; ++h) {      // sixteen lanes of the accumulator in v, sixteen in u, eight apart
          const uint32_t* from = h < 2 ? v : u;
          uint8_t* to = buf + (8 * j + 2 * (lane & 3)) * P + (q4 * 32 + 8 * h + (lane >> 2)) * 4;
          *reinterpret_cast<uint32_t*>(to) = from[4 * j + 2 * (h & 1)];
          *reinterpret_cast<uint32_t*>(to + P) = from[4 * j + 2 * (h & 1) + 1];
        }
      named_bar_sync(bar, 128);
      const int n = n0 + lane * 4;
      if (n < N) {
        float* dst = out.y32 + static_cast<int64_t>(r0 + c) * N + n;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i * 4 + q4;
          if (c + row < live)
            *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(row) * N) = *reinterpret_cast<const uint4*>(buf + row * P + lane * 16);
        }
      }
    } else if constexpr (EPI == kStore) {
      uint32_t w[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          w[j][h] = pack_bf16x2(__uint_as_float(v[4 * j + 2 * h]), __uint_as_float(v[4 * j + 2 * h + 1]));
          w[j][2 + h] = pack_bf16x2(__uint_as_float(u[4 * j + 2 * h]), __uint_as_float(u[4 * j + 2 * h + 1]));
        }
      named_bar_sync(bar, 128);      // the rows staged before have been read
#pragma unroll
      for (int j = 0; j < 4; ++j) stmatrix_x4_trans(put + j * 8 * P, w[j][0], w[j][1], w[j][2], w[j][3]);
      named_bar_sync(bar, 128);
      const int n = n0 + (tid & 15) * 8;
      if (n < N) {
        __nv_bfloat16* dst = out.y + static_cast<int64_t>(r0 + c) * N + n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = i * 8 + (tid >> 4);
          if (c + row < live)
            *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(row) * N) = *reinterpret_cast<const uint4*>(buf + row * P + (tid & 15) * 16);
        }
      }
    } else {
      const int f0 = n0 + q4 * 16;
      const bool in0 = f0 < N, in1 = f0 + 8 < N;      // units of a fragment's two halves
      uint32_t act[4][2], gate[4][2], up[4][2];       // pairs of neighbouring output rows
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float g0 = __uint_as_float(v[4 * j + 2 * h]), g1 = __uint_as_float(v[4 * j + 2 * h + 1]);
          const float u0 = __uint_as_float(u[4 * j + 2 * h]), u1 = __uint_as_float(u[4 * j + 2 * h + 1]);
          act[j][h] = pack_bf16x2(silu(g0) * u0, silu(g1) * u1);
          const bool in = h ? in1 : in0;
          gate[j][h] = in ? pack_bf16x2(g0, g1) : 0u;
          up[j][h] = in ? pack_bf16x2(u0, u1) : 0u;
        }
      if constexpr (EPI == kSwiglu8) {
        uint32_t* tops = reinterpret_cast<uint32_t*>(buf + EPI_ROWS * P);                   // [warp][gate, up][32 rows] bf16
        float* inv = reinterpret_cast<float*>(buf + EPI_ROWS * P + MAX_BYTES);              // [gate, up][32 rows]
        const int nb = (N + kActBlock - 1) / kActBlock;
        // the largest magnitude of every row's 16 units: eight values over eight lanes, half of what is left handed on in each step
        uint32_t m[8];
        constexpr uint32_t kAbs = 0x7fff7fffu;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m[2 * j] = max2_nan(gate[j][0] & kAbs, gate[j][1] & kAbs);
          m[2 * j + 1] = max2_nan(up[j][0] & kAbs, up[j][1] & kAbs);
        }
#pragma unroll
        for (int bit = 16, n = 4; bit >= 4; bit >>= 1, n >>= 1)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < n) {
              const uint32_t give = (lane & bit) ? m[i] : m[i + n], keep = (lane & bit) ? m[i + n] : m[i];
              m[i] = max2_nan(keep, __shfl_xor_sync(0xffffffffu, give, bit));
            }
        const int j0 = (lane >> 4) * 2 + ((lane >> 3) & 1), half0 = (lane >> 2) & 1;
        tops[q4 * 32 + half0 * 16 + j0 * 4 + (lane & 3)] = m[0];
        named_bar_sync(bar, 128);      // (also: the rows staged before have been read)
        if (q4 < 2) {      // a thread has the gates or the ups of one row
          float a = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float t = __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(tops)[w * 64 + q4 * 32 + lane]) << 16);
            a = t != t ? t : (a != a ? a : fmaxf(a, t));
          }
          const ActScale k = act_scale(a);
          inv[q4 * 32 + lane] = k.inv;
          const int blk = n0 / kActBlock;
          if (c + lane < live && blk < nb) out.scales[static_cast<int64_t>(r0 + c + lane) * 2 * nb + q4 * nb + blk] = k.scale;
        }
        named_bar_sync(bar, 128);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 ig = *reinterpret_cast<const float2*>(inv + 8 * j + 2 * (lane & 3));
          const float2 iu = *reinterpret_cast<const float2*>(inv + 32 + 8 * j + 2 * (lane & 3));
          uint8_t* to = buf + (8 * j + 2 * (lane & 3)) * P + 128 + q4 * 16 + (lane >> 2);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            to[8 * h] = act_byte(__uint_as_float(gate[j][h] << 16), ig.x);
            to[P + 8 * h] = act_byte(__uint_as_float(gate[j][h] & 0xffff0000u), ig.y);
            to[64 + 8 * h] = act_byte(__uint_as_float(up[j][h] << 16), iu.x);
            to[P + 64 + 8 * h] = act_byte(__uint_as_float(up[j][h] & 0xffff0000u), iu.y);
          }
        }
      } else {
        named_bar_sync(bar, 128);      // the rows staged before have been read
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        stmatrix_x2_trans(put + j * 8 * P, act[j][0], act[j][1]);
        if constexpr (EPI == kSwiglu) {
          stmatrix_x2_trans(put + j * 8 * P + 128, gate[j][0], gate[j][1]);
          stmatrix_x2_trans(put + j * 8 * P + 256, up[j][0], up[j][1]);
        }
      }
      named_bar_sync(bar, 128);
      const int piece = tid & 7, n = n0 + piece * 8;
      if (n < N) {
        const int64_t at = static_cast<int64_t>(r0 + c);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = i * 16 + (tid >> 3);
          if (c + row < live) {
            const uint8_t* src = buf + row * P;
            *reinterpret_cast<uint4*>(out.y + (at + row) * N + n) = *reinterpret_cast<const uint4*>(src + piece * 16);
            if constexpr (EPI == kSwiglu) {
              if (out.gu) {
                __nv_bfloat16* gu = out.gu + (at + row) * 2 * N + n;
                *reinterpret_cast<uint4*>(gu) = *reinterpret_cast<const uint4*>(src + 128 + piece * 16);
                *reinterpret_cast<uint4*>(gu + N) = *reinterpret_cast<const uint4*>(src + 256 + piece * 16);
              }
            } else {
              int8_t* q = out.q + (at + row) * 2 * N + n;
              *reinterpret_cast<uint2*>(q) = *reinterpret_cast<const uint2*>(src + 128 + piece * 8);
              *reinterpret_cast<uint2*>(q + N) = *reinterpret_cast<const uint2*>(src + 192 + piece * 8);
            }
          }
        }
      }
    }
  }
}

// Zeros into the rows of no expert, by `warps` warps of which this is number `w`
template <int EPI>
__device__ __forceinline__ void rows_of_none(const RowsOut& out, int first, int R, int w, int warps) {
  const int lane = threadIdx.x & 31, N = out.width;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int r = first + w; r < R; r += warps) {
    const int64_t row = r;
    if (EPI == kStore32) {
      for (int n = lane * 4; n < N; n += 128) *reinterpret_cast<uint4*>(out.y32 + row * N + n) = zero;
      continue;
    }
    for (int n = lane * 8; n < N; n += 256) *reinterpret_cast<uint4*>(out.y + row * N + n) = zero;
    if (EPI == kSwiglu && out.gu)
      for (int n = lane * 8; n < 2 * N; n += 256) *reinterpret_cast<uint4*>(out.gu + row * 2 * N + n) = zero;
    if (EPI == kSwiglu8) {
      const int nb = (N + kActBlock - 1) / kActBlock;
      for (int n = lane * 8; n < 2 * N; n += 256) *reinterpret_cast<uint2*>(out.q + row * 2 * N + n) = make_uint2(0, 0);
      for (int b = lane; b < 2 * nb; b += 32) out.scales[row * 2 * nb + b] = 0.f;
    }
  }
}

// The matrix's part of one k-block: 128 tile rows, from row (unit) n0 of expert e on.  Loads is FewLoads or PairLoads: where a copy
// is counted.
struct FewLoads {
  uint64_t* bar;
  __device__ __forceinline__ void d3(void* to, const CUtensorMap* m, int a, int b, int c) const { tma_load_3d(to, m, bar, a, b, c); }
  __device__ __forceinline__ void d4(void* to, const CUtensorMap* m, int a, int b, int c, int d) const { tma_load_4d(to, m, bar, a, b, c, d); }
  __device__ __forceinline__ void d5(void* to, const CUtensorMap* m, int a, int b, int c, int d, int e) const {
    tma_load_5d(to, m, bar, a, b, c, d, e);
  }
};
struct PairLoads {
  uint32_t bar;
  __device__ __forceinline__ void d3(void* to, const CUtensorMap* m, int a, int b, int c) const { tma_load_3d_pair(to, m, bar, a, b, c); }
  __device__ __forceinline__ void d4(void* to, const CUtensorMap* m, int a, int b, int c, int d) const {
    tma_load_4d_pair(to, m, bar, a, b, c, d);
  }
  __device__ __forceinline__ void d5(void* to, const CUtensorMap* m, int a, int b, int c, int d, int e) const {
    tma_load_5d_pair(to, m, bar, a, b, c, d, e);
  }
};
template <bool W_MN, int EPI, class Loads>
__device__ __forceinline__ void load_matrix(uint8_t* sA, const CUtensorMap* m, const RowsOut& out, int k0, int n0, int e, const Loads& loads) {
  if constexpr (kGateUp<EPI>) {
    if (out.width % 16 == 0) {
      loads.d5(sA, m, k0, 0, 0, n0 / 16, e);
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g) loads.d4(sA + g * 4096, m, k0, n0 + g * 16, 0, e);
    }
  } else if constexpr (W_MN) {
#pragma unroll
    for (int j = 0; j < BM / 64; ++j) loads.d3(sA + j * 8192, m, n0 + j * 64, k0, e);
  } else {
    loads.d3(sA, m, k0, n0, e);
  }
}

// y [R, N] from x [R, K] and matrices [E, N, K] (W_MN false) or [E, K, N]
template <bool W_MN, int EPI>
__global__ void __launch_bounds__(ROW_THREADS, 1)
grouped_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const int* __restrict__ offsets,
                    const __grid_constant__ RowsOut out, int R, int E, int K, int* err) {
  constexpr int UNIT = kGateUp<EPI> ? BM : 2 * BM;      // output columns of a tile
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* epi = smem + STAGES * STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi + ROW_EPI_BYTES);
  uint64_t* full = bars;                     // [STAGES]  used in the leader
  uint64_t* empty = bars + STAGES;           // [STAGES]  one per CTA
  uint64_t* tfull = bars + 2 * STAGES;       // [2]       one per CTA
  uint64_t* tempty = bars + 2 * STAGES + 2;  // [2]       used in the leader
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
  int* edge = reinterpret_cast<int*>(epi + ROW_EPI_BYTES + BAR_BYTES);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster = static_cast<int>(blockIdx.x) >> 1, num_clusters = static_cast<int>(gridDim.x) >> 1;
  const int cols = (out.width + UNIT - 1) / UNIT;
  const int num_kb = (K + BK - 1) / BK;

  load_edges(offsets, edge, E, R);
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 512);      // the epilogue threads of both CTAs
    }
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  Place at{edge, E, cols};

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0, r0, live, col;
      uint32_t phase = 0;
      bool ok = true;
      uint32_t lead_full[STAGES];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) lead_full[s] = map_to_cta(&full[s], 0);
      for (int n = cluster; ok && at.find(n, r0, live, col); n += num_clusters) {
        const int n0 = col * UNIT + static_cast<int>(rank) * (UNIT / 2);
        const int half = (live + 31) / 32 * 16;      // rows in each CTA's half of the instruction's columns
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, err, kErrProducerEmptyWait)) { ok = false; break; }
          uint8_t* sA = smem + stage * STAGE_BYTES;
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * STAGE_BYTES);
          load_matrix<W_MN, EPI>(sA, &tmW, out, kb * BK, n0, at.e, PairLoads{lead_full[stage]});
          tma_load_2d_pair(sA + A_BYTES, &tmX, lead_full[stage], kb * BK, r0 + static_cast<int>(rank) * half);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t a_lbo = W_MN ? 8192u : 16u, a_step = W_MN ? (2048u >> 4) : (32u >> 4);
      int stage = 0, it = 0, r0, live, col;
      uint32_t phase = 0;
      bool ok = true;
      for (int n = cluster; ok && at.find(n, r0, live, col); n += num_clusters) {
        const uint32_t idesc = make_idesc_bf16(2 * BM, (live + 31) / 32 * 32, W_MN, false);
        const int acc = it & 1;
        if (!mbar_wait(&tempty[acc], ((it >> 1) & 1) ^ 1, err, kErrMmaTmemEmptyWait)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, err, kErrMmaFullWait)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + stage * STAGE_BYTES);
          const uint64_t da = make_desc_sw128(a_addr, a_lbo, 1024);
          const uint64_t db = make_desc_sw128(a_addr + A_BYTES, 16u, 1024);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma2_f16_ss(d_tmem, da + static_cast<uint64_t>(k * a_step), db + static_cast<uint64_t>(k * (32u >> 4)), idesc,
                         (kb != 0 || k != 0) ? 1u : 0u);
          umma2_commit_both(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok) umma2_commit_both(&tfull[acc]);
        ++it;
      }
    }
  } else {
    const int q = warp & 3;                // TMEM lane quarter this warp may read
    const int part = (warp - 2) >> 2;      // two warps to a quarter, every other 32 columns each
    int it = 0, r0, live, col;
    bool ok = true;
    for (int n = cluster; ok && at.find(n, r0, live, col); n += num_clusters) {
      const int n0 = col * UNIT + static_cast<int>(rank) * (UNIT / 2);
      const int acc = it & 1;
      if (!mbar_wait_warps(&tfull[acc], (it >> 1) & 1, err, kErrEpilogueTmemFullWait, 1 + part, 128)) { ok = false; break; }
      tc_fence_after();
      const uint32_t lead_tempty = map_to_cta(&tempty[acc], 0);
      rows_epilogue<EPI>(out, tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN, q, epi + part * kPartBytes<EPI>, 1 + part, r0,
                         live, part * EPI_ROWS, 2 * EPI_ROWS, n0, [&] {
                           tc_fence_before();
                           pair_arrive(lead_tempty);      // (a release at cluster scope would wait for the rows sent to memory before)
                         });
      ++it;
    }
    rows_of_none<EPI>(out, edge[E], R, static_cast<int>(blockIdx.x) * 8 + warp - 2, static_cast<int>(gridDim.x) * 8);
  }

  if (*reinterpret_cast<volatile int*>(err) != 0) {
    // a wait expired somewhere: give copies and MMAs in flight time to land before TMEM is released
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// Few rows per group: one CTA has 128 tile rows (64 units of SwiGLU) of one group and up to 64 of its rows; grid (tiles of the matrix,
// an upper bound of the groups' tiles of rows).  The operand stages hold the epilogue's staging rows once the products are done.
// EARLY: the matrices are read before the kernel before has ended, which must not write them.  (A template, since the few instructions cost
// grids of a thousand CTAs 3 % where they are not used.)
constexpr int FEW_ROWS = 64, FEW_STAGES = 4, FEW_STAGE = A_BYTES + FEW_ROWS * BK * 2;
constexpr int FEW_SMEM = FEW_STAGES * FEW_STAGE + BAR_BYTES + 1024;
static_assert(ROW_EPI_BYTES <= FEW_STAGES * FEW_STAGE && kPartBytes<kStore32> <= FEW_STAGES * FEW_STAGE, "staging rows");
static_assert(2 * (FEW_SMEM + 1024) <= 233472, "two CTAs on an SM");

template <bool W_MN, int EPI, bool LISTED, bool EARLY>
__global__ void __launch_bounds__(FEW_THREADS, 2)
grouped_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const int* __restrict__ offsets,
                   const __grid_constant__ Rows rows, const __grid_constant__ RowsOut out, int R, int E, int K, int* err) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + FEW_STAGES * FEW_STAGE);
  uint64_t* full = bars;
  uint64_t* empty = bars + FEW_STAGES;
  uint64_t* tfull = bars + 2 * FEW_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * FEW_STAGES + 1);
  int* where = reinterpret_cast<int*>(bars + 2 * FEW_STAGES + 2);      // group, first row, rows, first row of no expert

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int UNIT = kGateUp<EPI> ? BM / 2 : BM;
  const int n0 = static_cast<int>(blockIdx.x) * UNIT, all_kb = (K + BK - 1) / BK;
  const int early = EARLY ? E : 0;
  const int loaded = static_cast<int>(blockIdx.y) < early ? min(all_kb, FEW_STAGES) : 0;      // k-blocks of the matrix under way
  if (warp == 1) {      // (warp 0 looks for its rows meanwhile)
    if (elect_one()) {
      tma_prefetch_desc(&tmW);
      tma_prefetch_desc(&tmX);
      for (int s = 0; s < FEW_STAGES; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], 1);
      }
      mbar_init(tfull, 1);
      fence_barrier_init();
      for (int kb = 0; kb < loaded; ++kb) {
        mbar_expect_more(&full[kb], A_BYTES);
        load_matrix<W_MN, EPI>(smem + kb * FEW_STAGE, &tmW, out, kb * BK, n0, blockIdx.y, FewLoads{&full[kb]});
      }
    }
    __syncwarp();
    tmem_alloc(tmem_slot, FEW_ROWS);
    tmem_relinquish();
    tc_fence_before();
  }
  pdl_wait();
  pdl_launch_dependents();
  if (warp == 0) {
    // the group that tile blockIdx.y of the groups' row tiles belongs to: edges as load_edges has them, 32 groups at a time.  With EARLY
    // the first tile of each group has a place of its own, and the others follow.
    int run = 0, tiles_before = early;
    if (lane == 0) where[2] = 0;
    __syncwarp();
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      int hi = e < E ? min(max(offsets[e + 1], 0), R) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, hi, o);
        if (lane >= o) hi = max(hi, up);
      }
      hi = max(hi, run);
      int lo = __shfl_up_sync(0xffffffffu, hi, 1);
      if (lane == 0) lo = run;
      const int placed = e < early && hi > lo ? 1 : 0, tiles = (hi - lo + FEW_ROWS - 1) / FEW_ROWS - placed;
      int sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      int at = static_cast<int>(blockIdx.y) - (tiles_before + sum - tiles);
      const bool mine = placed && e == static_cast<int>(blockIdx.y);
      if (mine || (at >= 0 && at < tiles)) {
        at = mine ? 0 : at + placed;
        where[0] = e;
        where[1] = lo + at * FEW_ROWS;
        where[2] = min(FEW_ROWS, hi - lo - at * FEW_ROWS);
      }
      run = __shfl_sync(0xffffffffu, hi, 31);
      tiles_before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) where[3] = run;
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const int e = where[0], r0 = where[1], live = where[2];
  const int num_kb = live > 0 ? all_kb : 0;

  if (warp == 0 && num_kb == 0) {      // what was asked for arrives before the CTA goes
    if (elect_one())
      for (int kb = 0; kb < loaded; ++kb) {
        mbar_arrive(&full[kb]);
        if (!mbar_wait(&full[kb], 0, err, kErrMmaFullWait)) break;
      }
    __syncwarp();
  }

  if (LISTED && warp == 0) {
    // all lanes: each has four of the rows; the first matrix tiles are on their way before the list is looked at
    int stage = 0;
    uint32_t phase = 0;
    const int used = (live + 15) / 16 * 16, ahead = min(num_kb, FEW_STAGES);
    if (lane == 0)
      for (int kb = 0; kb < ahead; ++kb) {
        mbar_expect_tx(&full[kb], (kb < loaded ? 0 : A_BYTES) + used * 128);
        if (kb >= loaded) load_matrix<W_MN, EPI>(smem + kb * FEW_STAGE, &tmW, out, kb * BK, n0, e, FewLoads{&full[kb]});
      }
    __syncwarp();
    int from[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) from[i] = num_kb > 0 ? rows.at(r0 + 4 * lane + i, r0 + live) : 0;
    for (int kb = 0; kb < num_kb; ++kb) {
      if (!mbar_wait_warp(&empty[stage], phase ^ 1, err, kErrProducerEmptyWait)) break;
      uint8_t* sA = smem + stage * FEW_STAGE;
      if (lane == 0 && kb >= ahead) {
        mbar_expect_tx(&full[stage], A_BYTES + used * 128);
        load_matrix<W_MN, EPI>(sA, &tmW, out, kb * BK, n0, e, FewLoads{&full[stage]});
      }
      if (4 * lane < used) tma_gather4(sA + A_BYTES + lane * 512, &tmX, &full[stage], kb * BK, from);
      if (++stage == FEW_STAGES) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, err, kErrProducerEmptyWait)) break;
        uint8_t* sA = smem + stage * FEW_STAGE;
        mbar_expect_tx(&full[stage], kb < loaded ? FEW_STAGE - A_BYTES : FEW_STAGE);
        if (kb >= loaded) load_matrix<W_MN, EPI>(sA, &tmW, out, kb * BK, n0, e, FewLoads{&full[stage]});
        tma_load_2d(sA + A_BYTES, &tmX, &full[stage], kb * BK, r0);
        if (++stage == FEW_STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t a_lbo = W_MN ? 8192u : 16u, a_step = W_MN ? (2048u >> 4) : (32u >> 4);
      const uint32_t idesc = make_idesc_bf16(BM, (live + 15) / 16 * 16, W_MN, false);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&full[stage], phase, err, kErrMmaFullWait)) { ok = false; break; }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(smem + stage * FEW_STAGE);
        const uint64_t da = make_desc_sw128(a_addr, a_lbo, 1024);
        const uint64_t db = make_desc_sw128(a_addr + A_BYTES, 16u, 1024);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          umma_f16_ss(tmem_base, da + static_cast<uint64_t>(k * a_step), db + static_cast<uint64_t>(k * (32u >> 4)), idesc,
                      (kb != 0 || k != 0) ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == FEW_STAGES) { stage = 0; phase ^= 1; }
      }
      if (ok && num_kb > 0) umma_commit(tfull);
    }
  } else {
    const int q = warp & 3;
    if (num_kb > 0 && mbar_wait_warps(tfull, 0, err, kErrEpilogueTmemFullWait, 1, 128)) {
      tc_fence_after();
      rows_epilogue<EPI>(out, tmem_base + (static_cast<uint32_t>(q * 32) << 16), q, smem, 1, r0, live, 0, EPI_ROWS, n0, [] {});
    }
    rows_of_none<EPI>(out, where[3], R, static_cast<int>(blockIdx.y * gridDim.x + blockIdx.x) * 4 + q,
                      static_cast<int>(gridDim.x * gridDim.y) * 4);
  }

  if (*reinterpret_cast<volatile int*>(err) != 0) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, FEW_ROWS);
  }
}

// Which tile of dw unit n is: the groups in falling order of their rows, so that what a pair takes last is short.  Eight groups of 16384
// rows, the largest five times the smallest: 51 instead of 57 us.
struct Tiles {
  const uint8_t* order;      // nullptr: as they come
  int per, num_n;
  __device__ __forceinline__ void at(int n, int& e, int& n0, int& k0) const {
    const int t = n % per;
    e = order ? order[n / per] : n / per;
    n0 = t % num_n * 2 * BM;
    k0 = t / num_n * BN;
  }
};

// dw [E, N, K], OUT 0: bf16, 1: fp32
template <int OUT>
__global__ void __launch_bounds__(W_THREADS, 1)
grouped_wgrad_kernel(const __grid_constant__ CUtensorMap tmDy, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmDw,
                     const int* __restrict__ offsets, int R, int E, int N, int K, int* err) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* epi = smem + STAGES * STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi + W_EPI_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* tail = bars + 2 * STAGES;        // [STAGES]  one per CTA: a block that needs rows zeroed has arrived here
  uint64_t* mended = bars + 3 * STAGES;      // [STAGES]  used in the leader: the partner has zeroed its rows
  uint64_t* tfull = bars + 4 * STAGES;
  uint64_t* tempty = bars + 4 * STAGES + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 * STAGES + 4);
  static_assert((4 * STAGES + 5) * 8 <= BAR_BYTES, "barriers");
  int* edge = reinterpret_cast<int*>(epi + W_EPI_BYTES + BAR_BYTES);
  uint8_t* order = reinterpret_cast<uint8_t*>(edge + kMaxExperts + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster = static_cast<int>(blockIdx.x) >> 1, num_clusters = static_cast<int>(gridDim.x) >> 1;
  const int num_n = (N + 2 * BM - 1) / (2 * BM), per = num_n * ((K + BN - 1) / BN), num_units = per * E;
  const Tiles tiles{E <= ORDERED ? order : nullptr, per, num_n};
  int e, n0, k0;

  load_edges(offsets, edge, E, R);
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tmDy);
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmDw);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tail[s], 1);
      mbar_init(&mended[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 512);
    }
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tc_fence_before();
  }
  __syncthreads();
  for (int a = threadIdx.x; a < E && E <= ORDERED; a += W_THREADS) {
    const int rows = edge[a + 1] - edge[a];
    int before = 0;
    for (int b = 0; b < E; ++b) {
      const int other = edge[b + 1] - edge[b];
      before += other > rows || (other == rows && b < a) ? 1 : 0;
    }
    order[before] = static_cast<uint8_t>(a);
  }
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      uint32_t lead_full[STAGES];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) lead_full[s] = map_to_cta(&full[s], 0);
      for (int n = cluster; n < num_units && ok; n += num_clusters) {
        tiles.at(n, e, n0, k0);
        const int lo = edge[e], rows = edge[e + 1] - lo;
        n0 += static_cast<int>(rank) * BM;
        k0 += static_cast<int>(rank) * BNH;
        const int num_kb = (rows + BK - 1) / BK;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, err, kErrProducerEmptyWait)) { ok = false; break; }
          uint8_t* sA = smem + stage * STAGE_BYTES;
          uint8_t* sB = sA + A_BYTES;
          const int r0 = lo + kb * BK;
          if (kb == num_kb - 1 && rows % 16 != 0) {
            mbar_expect_tx(&tail[stage], STAGE_BYTES);
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_2d(sA + j * 8192, &tmDy, &tail[stage], n0 + j * 64, r0);
#pragma unroll
            for (int j = 0; j < BNH / 64; ++j) tma_load_2d(sB + j * 8192, &tmX, &tail[stage], k0 + j * 64, r0);
          } else {
            if (rank == 0) mbar_expect_tx(&full[stage], 2 * STAGE_BYTES);
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_2d_pair(sA + j * 8192, &tmDy, lead_full[stage], n0 + j * 64, r0);
#pragma unroll
            for (int j = 0; j < BNH / 64; ++j) tma_load_2d_pair(sB + j * 8192, &tmX, lead_full[stage], k0 + j * 64, r0);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int n = cluster; n < num_units && ok; n += num_clusters) {
        tiles.at(n, e, n0, k0);
        const int rows = edge[e + 1] - edge[e];
        if (rows == 0) continue;
        constexpr uint32_t idesc = make_idesc_bf16(2 * BM, BN, true, true);
        const int acc = it & 1;
        if (!mbar_wait(&tempty[acc], ((it >> 1) & 1) ^ 1, err, kErrMmaTmemEmptyWait)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        const int num_kb = (rows + BK - 1) / BK;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, err, kErrMmaFullWait)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + stage * STAGE_BYTES);
          const uint64_t da = make_desc_sw128(a_addr, 8192u, 1024);
          const uint64_t db = make_desc_sw128(a_addr + A_BYTES, 8192u, 1024);
          const int steps = min(BK / 16, (rows - kb * BK + 15) / 16);
          for (int k = 0; k < steps; ++k)
            umma2_f16_ss(d_tmem, da + static_cast<uint64_t>(k * (2048u >> 4)), db + static_cast<uint64_t>(k * (2048u >> 4)), idesc,
                         (kb != 0 || k != 0) ? 1u : 0u);
          umma2_commit_both(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok) umma2_commit_both(&tfull[acc]);
        ++it;
      }
    }
  } else if (warp == 10) {
    // zeros into the rows of the next group in a last block
    int blocks = 0;                    // loaded so far, of all groups
    uint32_t tail_phase = 0, mended_phase = 0;      // a bit per stage
    bool ok = true;
    for (int n = cluster; n < num_units && ok; n += num_clusters) {
      tiles.at(n, e, n0, k0);
      const int rows = edge[e + 1] - edge[e];
      blocks += (rows + BK - 1) / BK;
      if (rows % 16 == 0) continue;
      const int stage = (blocks - 1) % STAGES;
      ok = mbar_wait_warp(&tail[stage], (tail_phase >> stage) & 1, err, kErrMmaFullWait);
      if (!ok) break;
      tail_phase ^= 1u << stage;
      const int first = rows % BK, count = (16 - first % 16) * 8;      // 16-byte pieces of a box of 64 columns
      uint8_t* from = smem + stage * STAGE_BYTES + first * 128;
      for (int i = lane; i < 4 * count; i += 32)
        *reinterpret_cast<uint4*>(from + (i / count) * 8192 + (i % count) * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (rank != 0) {
        if (lane == 0) remote_arrive(map_to_cta(&mended[stage], 0));
      } else {
        ok = mbar_wait_warp(&mended[stage], (mended_phase >> stage) & 1, err, kErrMmaFullWait);
        mended_phase ^= 1u << stage;
        if (ok && lane == 0) mbar_arrive(&full[stage]);
      }
      __syncwarp();
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;      // two warps to a quarter of the lanes, every other slab each
    uint8_t* buf = epi + (warp - 2) * EPI_BUF;
    constexpr int COLS = OUT == 0 ? 64 : 32;             // columns per staged slab (128 B per row)
    int it = 0;
    bool ok = true;
    for (int n = cluster; n < num_units && ok; n += num_clusters) {
      tiles.at(n, e, n0, k0);
      n0 += static_cast<int>(rank) * BM + q * 32;
      const bool some = edge[e + 1] > edge[e];
      const int acc = it & 1;
      if (some) {
        ok = mbar_wait_warp(&tfull[acc], (it >> 1) & 1, err, kErrEpilogueTmemFullWait);
        if (!ok) break;
        ++it;
      }
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN;
      const uint32_t lead_tempty = map_to_cta(&tempty[acc], 0);
#pragma unroll 1
      for (int c = part; c < BN / COLS; c += 2) {
        uint32_t v[64];
        __syncwarp();
        if (some) {
          tmem_ld_32x32b_x32(t_row + c * COLS, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
          if (OUT == 0) tmem_ld_32x32b_x32(t_row + c * COLS + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
          tmem_ld_wait();
          if (c == BN / COLS - 2 + part) {
            tc_fence_before();
            pair_arrive(lead_tempty);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = 0u;
        }
        if (n0 < N && k0 + c * COLS < K) {
          if (lane == 0) tma_wait_group_read<0>();      // the store that last used this buffer has read it
          __syncwarp();
          uint8_t* row = buf + lane * 128;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint4 pk;
            if (OUT == 0) {
              pk.x = pack_bf16x2(__uint_as_float(v[8 * j + 0]), __uint_as_float(v[8 * j + 1]));
              pk.y = pack_bf16x2(__uint_as_float(v[8 * j + 2]), __uint_as_float(v[8 * j + 3]));
              pk.z = pack_bf16x2(__uint_as_float(v[8 * j + 4]), __uint_as_float(v[8 * j + 5]));
              pk.w = pack_bf16x2(__uint_as_float(v[8 * j + 6]), __uint_as_float(v[8 * j + 7]));
            } else {
              pk.x = v[4 * j + 0]; pk.y = v[4 * j + 1]; pk.z = v[4 * j + 2]; pk.w = v[4 * j + 3];
            }
            *reinterpret_cast<uint4*>(row + ((j ^ (lane & 7)) << 4)) = pk;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&tmDw, buf, k0 + c * COLS, n0, e);
            tma_commit_group();
          }
        }
      }
    }
    if (lane == 0) tma_wait_group<0>();
  }

  if (*reinterpret_cast<volatile int*>(err) != 0) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// CTA pairs of a kernel that the current device holds at once (the two CTAs sit on the two SMs of one TPC), 0 if it cannot be told.  Asked once
// for each kernel and device; forward and backward passes launch from different threads.
int pairs_at_once(const void* kernel, cudaLaunchConfig_t cfg) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, int> found;
  int dev = 0, sms = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::lock_guard<std::mutex> lock(mu);
  int& kept = found[{kernel, dev}];
  if (kept > 0) return kept;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  cfg.gridDim = dim3(2 * (sms / 2));
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) return 0;
  return kept = n < sms / 2 ? n : sms / 2;
}

template <class... Params, class... Args>
int launch_pairs(void (*kern)(Params...), int threads, int smem, int64_t units, int num_sms, cudaStream_t stream, Args... args) {
  if (!ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem)) return -20;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int at_once = pairs_at_once(reinterpret_cast<const void*>(kern), cfg);
  if (at_once == 0) return -23;
  const int pairs = at_once < num_sms / 2 ? at_once : num_sms / 2;
  cfg.gridDim = dim3(2 * static_cast<int>(units < pairs ? units : pairs));
  cfg.stream = stream;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.numAttrs = 2;
  return launch_code(cudaLaunchKernelEx(&cfg, kern, args...));
}

}  // namespace

namespace {

// Up to this many rows per group, on average, the small tiles.  Small tiles, pairs, us back to back, products of 8 uneven groups (1024 x
// 1536), of 64 (1024 x 768): 32 rows per group 9.4, 10.0; 24.1, 26.2.  64 rows 9.9, 10.5; 26.7, 30.4.  96 rows 10.2, 11.1; 32.5, 32.2,
// but the whole feed-forward 46, 43.5; 118, 104.  The average counts experts without rows too (group sizes are on the device).  All rows
// with one expert, small tiles, pairs: 8 experts, 512 rows 6.8, 10.9; 64 experts, 2048 rows 9.0, 11.1, 4096 rows 14.2, 11.9.
constexpr int FEW_AVERAGE = 64;
// Between these averages a feed-forward's kernels ask for their matrices before they know their rows: with fewer rows many groups would
// have none, and with more the second tiles of groups, which come last, no longer find their matrices in L2.  The whole feed-forward without
// and with it, 16 experts of 1024 x 768: 4 rows 30.8, 29.4; 16 rows 31.8, 29.4; 32 rows 35.5, 34.7.  64 experts: 16 rows 80, 77; 32 rows 77.7,
// 75.6; 64 rows 100, 116.  (The rest of the tile into L2 as well gave nothing with 16 experts and cost 5 % with 64.)
constexpr int64_t EARLY_FROM = 2, EARLY_TO = 32;
// Up to this average the rows are gathered by the gate / up product itself.  Put in order before, gathered: 16 experts, 8 rows 30.1, 28.4; 16
// rows 30.8, 29.4; 24 rows 33.0, 33.0; 64 experts, 8 rows 71.4, 71.0; 16 rows 77.8, 77.8; 24 rows 73, 78.
constexpr int64_t LISTED_AVERAGE = 16;

template <bool W_MN, int EPI, bool LISTED>
int launch_few(const CUtensorMap& tw, const CUtensorMap& tx, const Rows& rows, const int* offsets, const RowsOut& out, int R, int E, int K,
               bool early, int* err, cudaStream_t stream) {
  constexpr int UNIT = kGateUp<EPI> ? BM / 2 : BM;
  // at most: every group with rows ends in a tile that is not full
  const auto launch = [&](auto kern, int groups) {
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(kern), FEW_SMEM)) return -20;
    const dim3 grid((out.width + UNIT - 1) / UNIT, R / FEW_ROWS + groups);
    return launch_code(launch_pdl(kern, grid, dim3(FEW_THREADS), FEW_SMEM, stream, tw, tx, offsets, rows, out, R, E, K, err));
  };
  if constexpr (EPI != kStore)
    if (early && R >= EARLY_FROM * E && R <= EARLY_TO * E) return launch(grouped_few_kernel<W_MN, EPI, LISTED, true>, E);
  return launch(grouped_few_kernel<W_MN, EPI, LISTED, false>, E < R ? E : R);
}

template <bool W_MN, int EPI>
int launch_rows(const __nv_bfloat16* x, int64_t ldx, const Rows& rows, const __nv_bfloat16* w, const int* offsets, const RowsOut& out, int R,
                int E, int K, bool early, int* err, int num_sms, cudaStream_t stream) {
  const int N = out.width;
  if (R < 1 || E < 1 || E > kMaxExperts || N < 1 || K < 1 || N % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(out.y) | reinterpret_cast<uintptr_t>(out.y32)) & 15) != 0)
    return -1;
  const bool few = R <= static_cast<int64_t>(FEW_AVERAGE) * E;
  if (rows.list && !(few && EPI == kSwiglu)) return -2;
  CUtensorMap tw, tx;
  int r = kGateUp<EPI> ? make_tmap_gate_up(&tw, w, E, N, K, N % 16 == 0 ? 4 : 1)
          : W_MN       ? make_tmap_3d(&tw, w, 2, E, K, N, 64, 64)
                       : make_tmap_3d(&tw, w, 2, E, N, K, BM, 64);
  if (r) return r;
  r = rows.list ? make_tmap_2d(&tx, x, 2, rows.count, K, ldx, 1, 64) : make_tmap_2d(&tx, x, 2, R, K, ldx, few ? FEW_ROWS : BNH, 64);
  if (r) return r - 100;
  if constexpr (EPI == kSwiglu)
    if (rows.list) return launch_few<W_MN, EPI, true>(tw, tx, rows, offsets, out, R, E, K, early, err, stream);
  if constexpr (EPI == kStore32) {
    return few ? launch_few<W_MN, EPI, false>(tw, tx, rows, offsets, out, R, E, K, early, err, stream) : -2;
  } else {
    if (few) return launch_few<W_MN, EPI, false>(tw, tx, rows, offsets, out, R, E, K, early, err, stream);
    constexpr int UNIT = kGateUp<EPI> ? BM : 2 * BM;
    const int64_t units = (static_cast<int64_t>(R) / BN + (E < R ? E : R)) * ((N + UNIT - 1) / UNIT);
    return launch_pairs(grouped_rows_kernel<W_MN, EPI>, ROW_THREADS, ROW_SMEM, units, num_sms, stream, tw, tx, offsets, out, R, E, K, err);
  }
}

}  // namespace

int grouped_gemm(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* w, bool w_t, const int* offsets, __nv_bfloat16* y, int R,
                 int E, int N, int K, int* err, int num_sms, cudaStream_t stream) {
  RowsOut out{};
  out.y = y;
  out.width = N;
  const Rows rows{nullptr, FastDiv(1), 0};
  return w_t ? launch_rows<true, kStore>(x, ldx, rows, w, offsets, out, R, E, K, false, err, num_sms, stream)
             : launch_rows<false, kStore>(x, ldx, rows, w, offsets, out, R, E, K, false, err, num_sms, stream);
}

bool grouped_gemm_few(int R, int E) { return R <= static_cast<int64_t>(FEW_AVERAGE) * E; }

int grouped_gemm_f32(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* w, const int* offsets, float* y, int R, int E, int N, int K,
                     bool early, int* err, int num_sms, cudaStream_t stream) {
  RowsOut out{};
  out.y32 = y;
  out.width = N;
  return launch_rows<false, kStore32>(x, ldx, Rows{nullptr, FastDiv(1), 0}, w, offsets, out, R, E, K, early, err, num_sms, stream);
}

bool grouped_swiglu_listed(int R, int E) { return R <= LISTED_AVERAGE * E; }

int grouped_swiglu(const __nv_bfloat16* x, int64_t ldx, const int* list, int k, int count, const __nv_bfloat16* w, const int* offsets,
                   __nv_bfloat16* act, __nv_bfloat16* gu, int8_t* q, float* scales, int R, int E, int F, int K, bool early, int* err,
                   int num_sms, cudaStream_t stream) {
  if (F % 8 != 0 || (gu && q) || ((reinterpret_cast<uintptr_t>(gu) | reinterpret_cast<uintptr_t>(q)) & 15) != 0) return -1;
  RowsOut out{act, gu, q, scales, F, nullptr};
  const Rows rows{list, FastDiv(list ? k : 1), count};
  return q ? launch_rows<false, kSwiglu8>(x, ldx, rows, w, offsets, out, R, E, K, early, err, num_sms, stream)
           : launch_rows<false, kSwiglu>(x, ldx, rows, w, offsets, out, R, E, K, early, err, num_sms, stream);
}

int grouped_wgrad(const __nv_bfloat16* dy, int64_t lddy, const __nv_bfloat16* x, int64_t ldx, const int* offsets, void* dw, bool dw_bf16,
                  int R, int E, int N, int K, int* err, int num_sms, cudaStream_t stream) {
  if (R < 1 || E < 1 || E > kMaxExperts || N < 1 || K < 1) return -1;
  CUtensorMap ty, tx, tw;
  int r = make_tmap_2d(&ty, dy, 2, R, N, lddy, 64, 64);
  if (r) return r;
  r = make_tmap_2d(&tx, x, 2, R, K, ldx, 64, 64);
  if (r) return r - 100;
  r = dw_bf16 ? make_tmap_3d(&tw, dw, 2, E, N, K, 32, 64) : make_tmap_3d(&tw, dw, 4, E, N, K, 32, 32);
  if (r) return r - 200;
  const int64_t units = static_cast<int64_t>(E) * ((N + 2 * BM - 1) / (2 * BM)) * ((K + BN - 1) / BN);
  if (units > (1ll << 30)) return -3;
  return dw_bf16 ? launch_pairs(grouped_wgrad_kernel<0>, W_THREADS, W_SMEM, units, num_sms, stream, ty, tx, tw, offsets, R, E, N, K, err)
                 : launch_pairs(grouped_wgrad_kernel<1>, W_THREADS, W_SMEM, units, num_sms, stream, ty, tx, tw, offsets, R, E, N, K, err);
}

}  // namespace tb
