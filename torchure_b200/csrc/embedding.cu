// Embedding lookup with a scale, and its gradient by sorted tokens.
//
//   out[t] = scale table[ids[t]],   dtable[v] = scale sum over t with ids[t] == v of dout[t]
//
// Gradient: the tokens are sorted by id, equal ids in token order (a counting sort, digits of up to 9 bits from the lowest on: every CTA counts the
// digits of a run of tokens, adds up the counts before its own and ranks its tokens; no atomics decide an order).  Chunks of the sorted list are
// then summed each by a CTA, a run of equal ids at a time, and a finished row is written once.  A run that goes on in the next chunk leaves its part
// in scratch memory, and a last kernel adds up the parts of such runs: however often one token occurs, its rows are read by many CTAs.
// The table's gradient is mostly rows of no token: they are zeroed by CTAs of the sorting kernels, whose own work fills few SMs.
//
// Bound by memory: V D values of the gradient to write, T D to read.
#include "common.cuh"
#include "embed_api.h"

namespace tb {

namespace {

constexpr int kThreads = 1024;      // of the sorting kernels
constexpr int kWarps = kThreads / 32;
constexpr int kDigit = 9;           // bits, at most
constexpr int kMaxChunks = 148;
constexpr int kSegThreads = 256;
constexpr int kSegChunks = 148 * 8;      // chunks of the sorted list, at most (about)
constexpr int kSegMin = 16;              // tokens of a chunk, at least

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16(x); }
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
}

template <class I>
__device__ __forceinline__ int64_t id_at(const I* ids, int64_t t) { return static_cast<int64_t>(ids[t]); }

// ---- lookup -------------------------------------------------------------------------------------------
// A row's columns go to gridDim.y CTAs of 4 columns a thread (VEC) or 1; blockIdx.x strides over the rows.
template <class I, class S, class O, bool VEC>
__global__ void __launch_bounds__(256)
embedding_rows_kernel(const I* __restrict__ ids, const S* __restrict__ table, int64_t ld, O* __restrict__ out, float scale, int64_t T, int64_t V,
                      int D) {
  pdl_wait();
  pdl_launch_dependents();
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * (VEC ? 4 : 1);
  if (col >= D) return;
#pragma unroll 4
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < T; t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
    const int64_t id = id_at(ids, t);
    const bool there = id >= 0 && id < V;
    const S* row = table + (there ? id : 0) * ld + col;
    if constexpr (VEC) {
      float x[4];
      load4(row, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = there ? x[j] * scale : __uint_as_float(0x7fffffffu);
      store4(out + t * D + col, x);
    } else {
      put(out + t * D + col, there ? to_f(*row) * scale : __uint_as_float(0x7fffffffu));
    }
  }
}

// ---- sorting ------------------------------------------------------------------------------------------
struct Zero {                // a part of the table's gradient that CTAs from `from` on fill with zeros, in 16-byte pieces and a tail
  char* base;
  int64_t lo, hi;            // bytes
  int from;
};

__device__ void fill_zero(const Zero& z) {
  const int64_t n = static_cast<int64_t>(gridDim.x - z.from) * blockDim.x, i0 = static_cast<int64_t>(blockIdx.x - z.from) * blockDim.x + threadIdx.x;
  const int64_t quads = (z.hi - z.lo) >> 4;
  uint4* p = reinterpret_cast<uint4*>(z.base + z.lo);
  for (int64_t i = i0; i < quads; i += n) p[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = z.lo + (quads << 4) + i0; i < z.hi; i += n) z.base[i] = 0;
}

struct SortArgs {
  int T, chunk;              // tokens, and those of a CTA
  int shift, bins;           // of this pass's digit
  int V, padding;
};

// The sort key of a token: V (behind all rows) where it adds nothing
template <class I>
__device__ __forceinline__ uint2 first_entry(const I* ids, int t, const SortArgs& a) {
  const int64_t id = id_at(ids, t);
  const bool live = id >= 0 && id < a.V && id != a.padding;
  return make_uint2(live ? static_cast<uint32_t>(id) : static_cast<uint32_t>(a.V), static_cast<uint32_t>(t));
}
struct FromIds32 { const int* p; __device__ uint2 operator()(int t, const SortArgs& a) const { return first_entry(p, t, a); } };
struct FromIds64 { const int64_t* p; __device__ uint2 operator()(int t, const SortArgs& a) const { return first_entry(p, t, a); } };
struct FromPass { const uint2* p; __device__ uint2 operator()(int t, const SortArgs&) const { return p[t]; } };

template <class From>
__global__ void __launch_bounds__(kThreads)
sort_count_kernel(From from, SortArgs a, int* __restrict__ hist, Zero z) {
  pdl_wait();
  pdl_launch_dependents();
  if (static_cast<int>(blockIdx.x) >= z.from) return fill_zero(z);
  __shared__ int count[1 << kDigit];
  for (int b = threadIdx.x; b < a.bins; b += kThreads) count[b] = 0;
  __syncthreads();
  const int lo = blockIdx.x * a.chunk, hi = min(a.T, lo + a.chunk);
  for (int t = lo + threadIdx.x; t < hi; t += kThreads) atomicAdd(&count[(from(t, a).x >> a.shift) & (a.bins - 1)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < a.bins; b += kThreads) hist[static_cast<int64_t>(blockIdx.x) * a.bins + b] = count[b];
}

// [kWarps][bins | 1] counts of the warps, and the first place of each bin for this CTA
constexpr int rank_smem(int bins) { return 4 * (kWarps * (bins | 1) + bins + kWarps); }

template <class From>
__global__ void __launch_bounds__(kThreads)
sort_rank_kernel(From from, SortArgs a, const int* __restrict__ hist, int chunks, uint2* __restrict__ out, Zero z) {
  pdl_wait();
  pdl_launch_dependents();
  if (static_cast<int>(blockIdx.x) >= z.from) return fill_zero(z);
  extern __shared__ int sm[];
  const int S = a.bins | 1, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = blockIdx.x;
  int* cnt = sm;                       // [kWarps][S]
  int* place = sm + kWarps * S;        // [bins]
  int* sums = place + a.bins;          // [kWarps]
  for (int i = tid; i < kWarps * S; i += kThreads) cnt[i] = 0;
  __syncthreads();
  // this CTA's tokens, a consecutive part for each warp
  const int lo = c * a.chunk, count = min(a.T - lo, a.chunk);
  const int part = ((count + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int wlo = min(count, warp * part), whi = min(count, wlo + part);
  for (int i = wlo + lane; i < whi; i += 32) atomicAdd(&cnt[warp * S + ((from(lo + i, a).x >> a.shift) & (a.bins - 1))], 1);
  // (bins are at most half the threads) counts of all CTAs, and of those before
  int all = 0, before = 0;
  if (tid < a.bins) {
#pragma unroll 8
    for (int i = 0; i < chunks; ++i) {
      const int v = hist[static_cast<int64_t>(i) * a.bins + tid];
      all += v;
      before += i < c ? v : 0;
    }
  }
  int up = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += v;
  }
  if (lane == 31) sums[warp] = up;
  __syncthreads();
  if (tid < a.bins) {
    int base = 0;
    for (int w = 0; w < warp; ++w) base += sums[w];
    place[tid] = base + up - all + before;
  }
  __syncthreads();
  for (int b = warp; b < a.bins; b += kWarps) {      // a lane per warp's count
    const int n = cnt[lane * S + b];
    int s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    cnt[lane * S + b] = place[b] + s - n;
  }
  __syncthreads();
  for (int i0 = wlo; i0 < whi; i0 += 32) {
    const int i = i0 + lane;
    const uint2 e = i < whi ? from(lo + i, a) : make_uint2(0, 0);
    const int b = i < whi ? static_cast<int>((e.x >> a.shift) & (a.bins - 1)) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, b);
    const int rank = __popc(same & ((1u << lane) - 1u));
    const int at = b >= 0 ? cnt[warp * S + b] + rank : 0;
    __syncwarp();
    if (b >= 0 && rank == 0) cnt[warp * S + b] += __popc(same);
    __syncwarp();
    if (b >= 0) out[at] = e;
  }
}

// ---- sums ---------------------------------------------------------------------------------------------
struct SumArgs {
  const uint2* sorted;       // (id, token), ids rising
  int T, chunk, V, D;
  int64_t ld;
  float scale;
  float* parts;              // [2 chunks][D]: what a chunk adds to the run that came in, and what it begins of the one that goes on
};

// A thread's four columns: next to each other (VEC) or a CTA's width apart
template <bool VEC, class T>
__device__ __forceinline__ void load_cols(const T* row, int col, int step, int D, float (&x)[4]) {
  if constexpr (VEC) {
    load4(row + col, x);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = col + j * step < D ? to_f(row[col + j * step]) : 0.f;
  }
}
template <bool VEC, class T>
__device__ __forceinline__ void store_cols(T* row, int col, int step, int D, const float (&x)[4]) {
  if constexpr (VEC) {
    store4(row + col, x);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j * step < D) put(row + col + j * step, x[j]);
  }
}

template <class S, class O, bool VEC>
__global__ void __launch_bounds__(kSegThreads)
segment_sum_kernel(SumArgs a, const S* __restrict__ dout, O* __restrict__ dtable) {
  pdl_wait();
  pdl_launch_dependents();
  const int step = blockDim.x, col = blockIdx.y * step * 4 + threadIdx.x * (VEC ? 4 : 1);
  const int lo = blockIdx.x * a.chunk, hi = min(a.T, lo + a.chunk);
  if (VEC && col >= a.D) return;
  const uint32_t none = static_cast<uint32_t>(a.V);
  const uint32_t came = lo > 0 ? a.sorted[lo - 1].x : none, goes = hi < a.T ? a.sorted[hi].x : none;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t run = a.sorted[lo].x;
  bool open = run == came;           // the run began before this chunk
  if (run == none) return;
  constexpr int U = 8;
  for (int i0 = lo; i0 < hi; i0 += U) {
    uint2 e[U];
    float x[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) e[u] = i0 + u < hi ? a.sorted[i0 + u] : make_uint2(none, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (e[u].x != none) load_cols<VEC>(dout + static_cast<int64_t>(e[u].y) * a.ld, col, step, a.D, x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (e[u].x != run) {
        if (open) {
          store_cols<VEC>(a.parts + static_cast<int64_t>(2 * blockIdx.x) * a.D, col, step, a.D, acc);
        } else if (run != none && !(i0 + u >= hi && run == goes)) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] *= a.scale;
          store_cols<VEC>(dtable + static_cast<int64_t>(run) * a.D, col, step, a.D, acc);
        } else if (run != none) {
          store_cols<VEC>(a.parts + static_cast<int64_t>(2 * blockIdx.x + 1) * a.D, col, step, a.D, acc);
        }
        if (e[u].x == none) return;
        run = e[u].x;
        open = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += x[u][j];
    }
  }
  // a chunk of a multiple of U tokens: its last run
  if (open) {
    store_cols<VEC>(a.parts + static_cast<int64_t>(2 * blockIdx.x) * a.D, col, step, a.D, acc);
  } else if (run == goes) {
    store_cols<VEC>(a.parts + static_cast<int64_t>(2 * blockIdx.x + 1) * a.D, col, step, a.D, acc);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] *= a.scale;
    store_cols<VEC>(dtable + static_cast<int64_t>(run) * a.D, col, step, a.D, acc);
  }
}

// Runs over several chunks, each by the CTAs of the chunk that it begins in: its part there, and those of the chunks up to its end
template <class O>
__global__ void __launch_bounds__(kSegThreads)
segment_join_kernel(SumArgs a, O* __restrict__ dtable) {
  pdl_wait();
  pdl_launch_dependents();
  const int c = blockIdx.x, lo = c * a.chunk, hi = min(a.T, lo + a.chunk);
  if (hi >= a.T) return;
  const uint32_t run = a.sorted[hi - 1].x;
  if (run == static_cast<uint32_t>(a.V) || a.sorted[hi].x != run || (lo > 0 && a.sorted[lo - 1].x == run)) return;
  int first = hi, last = a.T;              // the run ends before `last`
  while (first < last) {
    const int mid = first + (last - first) / 2;
    if (a.sorted[mid].x == run) first = mid + 1;
    else last = mid;
  }
  const int end = (first - 1) / a.chunk;   // its last chunk
  __shared__ float part[kSegThreads / 32][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y * 32 + lane;
  float s = 0.f;
  if (col < a.D) {
#pragma unroll 8
    for (int i = c + warp; i <= end; i += kSegThreads / 32) s += a.parts[static_cast<int64_t>(2 * i + (i == c ? 1 : 0)) * a.D + col];
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && col < a.D) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < kSegThreads / 32; ++w) s += part[w][lane];
    put(dtable + static_cast<int64_t>(run) * a.D + col, s * a.scale);
  }
}

int bits_of(int64_t n) {             // of the largest value below n
  int b = 1;
  while ((1ll << b) < n) ++b;
  return b;
}
struct Plan {
  int passes, bits, chunks, chunk, seg_chunk, seg_chunks;
};
Plan plan_for(int64_t T, int64_t V) {
  Plan p{};
  const int bits = bits_of(V + 1);
  p.passes = (bits + kDigit - 1) / kDigit;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.chunk = static_cast<int>((T + kMaxChunks - 1) / kMaxChunks);
  p.chunk = (p.chunk + kThreads - 1) / kThreads * kThreads;
  p.chunks = static_cast<int>((T + p.chunk - 1) / p.chunk);
  p.seg_chunk = static_cast<int>((T + kSegChunks - 1) / kSegChunks);
  p.seg_chunk = p.seg_chunk < kSegMin ? kSegMin : (p.seg_chunk + 7) / 8 * 8;
  p.seg_chunks = static_cast<int>((T + p.seg_chunk - 1) / p.seg_chunk);
  return p;
}
int64_t on16(int64_t n) { return (n + 15) / 16 * 16; }
bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <class I, class S, class O>
int launch_rows(const I* ids, const S* table, int64_t ld, O* out, float scale, int64_t T, int64_t V, int D, cudaStream_t stream) {
  const bool vec = D % 4 == 0 && ld % 4 == 0 && aligned(table, 4 * sizeof(S)) && aligned(out, 4 * sizeof(O));
  const int units = vec ? D / 4 : D;
  int width = 32;
  while (width < 256 && width < units) width *= 2;
  const dim3 block(width, 256 / width);
  const int64_t rows = (T + block.y - 1) / block.y;
  const dim3 grid(static_cast<unsigned>(rows < 148 * 32 ? rows : 148 * 32), (units + width - 1) / width);
  return launch_code(vec ? launch_pdl(embedding_rows_kernel<I, S, O, true>, grid, block, 0, stream, ids, table, ld, out, scale, T, V, D)
                         : launch_pdl(embedding_rows_kernel<I, S, O, false>, grid, block, 0, stream, ids, table, ld, out, scale, T, V, D));
}

template <class S, class O>
int launch_sums(const SumArgs& a, int chunks, const S* dout, O* dtable, cudaStream_t stream) {
  const bool vec = a.D % 4 == 0 && a.ld % 4 == 0 && aligned(dout, 4 * sizeof(S)) && aligned(dtable, 4 * sizeof(O));
  int width = 32;
  while (width < kSegThreads && width * 4 < a.D) width *= 2;
  const dim3 grid(chunks, (a.D + width * 4 - 1) / (width * 4));
  int rc = launch_code(vec ? launch_pdl(segment_sum_kernel<S, O, true>, grid, dim3(width), 0, stream, a, dout, dtable)
                           : launch_pdl(segment_sum_kernel<S, O, false>, grid, dim3(width), 0, stream, a, dout, dtable));
  if (rc == 0 && chunks > 1)
    rc = launch_code(launch_pdl(segment_join_kernel<O>, dim3(chunks, (a.D + 31) / 32), dim3(kSegThreads), 0, stream, a, dtable));
  return rc;
}

bool fits(int64_t T, int64_t V, int D) {
  return T >= 1 && T <= (1ll << 30) && V >= 1 && V <= (1ll << 30) && D >= 1 && D <= (1 << 20);
}

}  // namespace

int64_t embedding_scratch_bytes(int64_t T, int64_t V, int D) {
  const Plan p = plan_for(T, V);
  return 2 * on16(8 * T) + on16(4ll * p.chunks << p.bits) + 8ll * p.seg_chunks * D;
}

int embedding_grad_kernels(int64_t T, int64_t V) {
  const Plan p = plan_for(T, V);
  return 2 * p.passes + (p.seg_chunks > 1 ? 2 : 1);
}

int embedding_rows(const void* ids, bool ids64, const void* table, bool table16, int64_t ld, void* out, bool out16, float scale, int64_t T,
                   int64_t V, int D, cudaStream_t stream) {
  if (!fits(T, V, D)) return -1;
  const auto go = [&](auto* i) {
    const auto from = [&](auto* s) {
      return out16 ? launch_rows(i, s, ld, static_cast<__nv_bfloat16*>(out), scale, T, V, D, stream)
                   : launch_rows(i, s, ld, static_cast<float*>(out), scale, T, V, D, stream);
    };
    return table16 ? from(static_cast<const __nv_bfloat16*>(table)) : from(static_cast<const float*>(table));
  };
  return ids64 ? go(static_cast<const int64_t*>(ids)) : go(static_cast<const int*>(ids));
}

int embedding_grad(const void* ids, bool ids64, const void* dout, bool dout16, int64_t ld, void* dtable, bool dtable16, float scale,
                   int64_t padding, int64_t T, int64_t V, int D, void* scratch, cudaStream_t stream) {
  if (!fits(T, V, D) || padding < -1 || padding >= V || !aligned(dtable, 16) || !aligned(scratch, 16)) return -1;
  const Plan p = plan_for(T, V);
  char* at = static_cast<char*>(scratch);
  uint2* lists[2] = {reinterpret_cast<uint2*>(at), reinterpret_cast<uint2*>(at + on16(8 * T))};
  at += 2 * on16(8 * T);
  int* hist = reinterpret_cast<int*>(at);
  at += on16(4ll * p.chunks << p.bits);
  SortArgs a{};
  a.T = static_cast<int>(T); a.chunk = p.chunk; a.bins = 1 << p.bits; a.V = static_cast<int>(V); a.padding = static_cast<int>(padding);
  const int64_t bytes = V * D * (dtable16 ? 2 : 4);
  // each of the sorting kernels fills its share of the gradient
  const int kernels = 2 * p.passes;
  int64_t done = 0;
  Zero z{static_cast<char*>(dtable), 0, 0, p.chunks};
  const auto share = [&](int i) {
    z.lo = done;
    z.hi = done = i + 1 == kernels ? bytes : bytes * (i + 1) / kernels / 16 * 16;
    int64_t ctas = (z.hi - z.lo + 16 * kThreads * 4 - 1) / (16 * kThreads * 4);
    if (ctas > 148 * 2) ctas = 148 * 2;
    return static_cast<int>(ctas < 1 ? 1 : ctas);
  };
  const int smem = rank_smem(a.bins);
  const auto pass = [&](auto from, int i) {
    using From = decltype(from);
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(sort_rank_kernel<From>), smem)) return -20;
    a.shift = i * p.bits;
    int more = share(2 * i);
    int rc = launch_code(launch_pdl(sort_count_kernel<From>, dim3(p.chunks + more), dim3(kThreads), 0, stream, from, a, hist, z));
    if (rc) return rc;
    more = share(2 * i + 1);
    return launch_code(launch_pdl(sort_rank_kernel<From>, dim3(p.chunks + more), dim3(kThreads), static_cast<size_t>(smem), stream, from, a,
                                  hist, p.chunks, lists[i & 1], z));
  };
  for (int i = 0; i < p.passes; ++i) {
    const int rc = i > 0 ? pass(FromPass{lists[(i - 1) & 1]}, i)
                   : ids64 ? pass(FromIds64{static_cast<const int64_t*>(ids)}, i)
                           : pass(FromIds32{static_cast<const int*>(ids)}, i);
    if (rc) return rc;
  }
  SumArgs s{};
  s.sorted = lists[(p.passes - 1) & 1];
  s.T = a.T; s.chunk = p.seg_chunk; s.V = a.V; s.D = D; s.ld = ld; s.scale = scale;
  s.parts = reinterpret_cast<float*>(at);
  const auto sums = [&](auto* d) {
    return dtable16 ? launch_sums(s, p.seg_chunks, d, static_cast<__nv_bfloat16*>(dtable), stream)
                    : launch_sums(s, p.seg_chunks, d, static_cast<float*>(dtable), stream);
  };
  return dout16 ? sums(static_cast<const __nv_bfloat16*>(dout)) : sums(static_cast<const float*>(dout));
}

}  // namespace tb
