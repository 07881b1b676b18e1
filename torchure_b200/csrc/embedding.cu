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
// Bound by memory: V D values of the gradient to write, T D to read.  8192 tokens, a table of 151936 x 1024 in fp32: lookup 10.2 us (6.6 TB/s), sort
// and zeros 86 (7.2 TB/s of zeros), sums 12.7, runs over chunks 6.2; the whole pass 114, of which the bytes take 110 at copy bandwidth.  65521 tokens of
// 1003 columns in bf16, 30 % padding: 43, 28, 39, 12.  Few tokens: a chain of kernels of 3 - 5 us.
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
constexpr int kJoinCols = 128;           // columns of a CTA that joins parts

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

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
template <class I>
__device__ __forceinline__ int64_t id_at(const I* ids, int64_t t) { return static_cast<int64_t>(ids[t]); }

// ---- lookup -------------------------------------------------------------------------------------------
// A warp has kRowCols columns of a row (blockIdx.y says which), at addresses that are constants behind one base: four next to each other for a thread
// and round (kRowsFours), or one (kRowsOnes).  bf16 rows of an odd width or stride are read and written as 32-bit words all the same
// (kRowsPairs): pairs of columns as the output's words have them, put together from two neighbouring words where the table's lie one column off.
// The ids of the rows to come are on their way meanwhile.  65521 rows of 1003 columns 50 us by ones and 42.5 by pairs, 45 if rows of scale 1 were
// taken apart and put together too; 8192 rows of 1024 in fp32, by fours, 10.1 (6.6 TB/s).
constexpr int kRowCols = 512;
enum RowsBy { kRowsFours, kRowsOnes, kRowsPairs };

template <class I, class S, class O, RowsBy BY>
__global__ void __launch_bounds__(256)
embedding_rows_kernel(const I* __restrict__ ids, const S* __restrict__ table, int64_t ld, O* __restrict__ out, float scale, int64_t T, int64_t V,
                      int D) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int W = BY == kRowsFours ? 4 : BY == kRowsPairs ? 2 : 1, N = kRowCols / 32 / W;
  const int lane = threadIdx.x & 31, begin = blockIdx.y * kRowCols, end = min(D, begin + kRowCols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32);
  int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  int64_t next = t < T ? id_at(ids, t) : 0;
  for (; t < T; t += step) {
    const int64_t id = next;
    if (t + step < T) next = id_at(ids, t + step);
    const bool there = id >= 0 && id < V;
    const float by = there ? scale : __uint_as_float(0x7fffffffu);      // (an id outside the table: NaN times its first row)
    const S* from = table + (there ? id : 0) * ld;
    O* to = out + t * D;
    const auto ones = [&](int first, int last) {
      for (int c0 = first; c0 < last; c0 += 512) {
        S x[16];
#pragma unroll
        for (int n = 0; n < 16; ++n)
          if (c0 + lane + n * 32 < last) x[n] = from[c0 + lane + n * 32];
#pragma unroll
        for (int n = 0; n < 16; ++n)
          if (c0 + lane + n * 32 < last) put(to + c0 + lane + n * 32, to_f(x[n]) * by);
      }
    };
    if constexpr (BY == kRowsFours) {
      const int col = begin + lane * 4;
      const auto part = [&](auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        float x[N][4];
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (kWhole || col + n * 128 < end) load4(from + col + n * 128, x[n]);
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[n][j] *= by;
          if (kWhole || col + n * 128 < end) store4(to + col + n * 128, x[n]);
        }
      };
      if (end - begin == kRowCols) part(Yes{});
      else part(No{});
    } else if constexpr (BY == kRowsOnes) {
      ones(begin, end);
    } else {
      // (a last row's words could reach behind the table)
      if (!there || id + 1 == V) {
        ones(begin, end);
        continue;
      }
      const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(to + begin) >> 1) & 1;      // columns before the output's first word
      const int first = begin + lead, pairs = (end - first) / 2;
      const uintptr_t at = reinterpret_cast<uintptr_t>(from + first);
      const bool off = (at & 2) != 0;
      const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
      const int n_words = pairs + (off ? 1 : 0);
      uint32_t* put_words = reinterpret_cast<uint32_t*>(to + first);
      uint32_t x[N + 1];
#pragma unroll
      for (int n = 0; n <= N; ++n) x[n] = lane + n * 32 < n_words ? words[lane + n * 32] : 0u;
      if (lane == 0 && lead) put(to + begin, to_f(from[begin]) * by);
      if (lane == 1 && first + 2 * pairs < end) put(to + end - 1, to_f(from[end - 1]) * by);
      const auto emit = [&](auto shifted, auto scaled) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          uint32_t w = x[n];
          if (decltype(shifted)::value) w = __funnelshift_r(w, __shfl_sync(0xffffffffu, lane == 0 ? x[n + 1] : w, (lane + 1) & 31), 16);
          if (decltype(scaled)::value) w = pack_bf16x2(__uint_as_float(w << 16) * by, __uint_as_float(w & 0xffff0000u) * by);
          if (lane + n * 32 < pairs) put_words[lane + n * 32] = w;
        }
      };
      if (by == 1.f) off ? emit(Yes{}, No{}) : emit(No{}, No{});      // (a row as it is)
      else off ? emit(Yes{}, Yes{}) : emit(No{}, Yes{});
    }
  }
}

// ---- sorting ------------------------------------------------------------------------------------------
struct Zero {                // a part of the table's gradient that CTAs from `from` on fill with zeros, in 16-byte pieces and a tail
  char* base;
  int64_t lo, hi;            // bytes
  int from;
  int* spans;                // set to 0 too
};

__device__ void fill_zero(const Zero& z) {
  constexpr int kPiece = 4 * kThreads;      // 64 KB
  const int64_t ctas = gridDim.x - z.from, me = blockIdx.x - z.from, quads = (z.hi - z.lo) >> 4;
  uint4* p = reinterpret_cast<uint4*>(z.base + z.lo) + threadIdx.x;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int64_t q = me * kPiece; q < quads; q += ctas * kPiece) {
    const int64_t left = quads - q - threadIdx.x;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j * kThreads < left) p[q + j * kThreads] = zero;
  }
  if (me == 0 && threadIdx.x == 0) *z.spans = 0;
  if (me == 0 && threadIdx.x < ((z.hi - z.lo) & 15)) z.base[z.lo + (quads << 4) + threadIdx.x] = 0;
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
sort_count_kernel(From from, SortArgs a, int* __restrict__ hist) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ int count[1 << kDigit];
  for (int b = threadIdx.x; b < a.bins; b += kThreads) count[b] = 0;
  __syncthreads();
  const int lo = blockIdx.x * a.chunk, hi = min(a.T, lo + a.chunk);
  for (int t = lo + threadIdx.x; t < hi; t += kThreads) atomicAdd(&count[(from(t, a).x >> a.shift) & (a.bins - 1)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < a.bins; b += kThreads) hist[static_cast<int64_t>(blockIdx.x) * a.bins + b] = count[b];
}

// One stable counting sort of a CTA's tokens by a digit.  `entry(i)`: token i of `count`, in parts of consecutive ones for each warp;
// `others(bin)`: (tokens of this bin in all CTAs, in those before), or nothing but the own; `put(place, entry)` takes what was sorted.
// cnt [kWarps][bins | 1], place [bins], sums [kWarps]
constexpr int rank_ints(int bins) { return kWarps * (bins | 1) + bins + kWarps; }

template <class Entry, class Others, class Put>
__device__ __forceinline__ void sort_pass(int count, int shift, int bins, int* sm, Entry entry, Others others, Put put) {
  const int S = bins | 1, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;      // (odd: the counts of a bin lie in different banks)
  int* cnt = sm;
  int* place = sm + kWarps * S;
  int* sums = place + bins;
  for (int i = tid; i < kWarps * S; i += kThreads) cnt[i] = 0;
  __syncthreads();
  const int part = ((count + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int lo = min(count, warp * part), hi = min(count, lo + part);
  constexpr int U = 8;                              // entries of a thread that are on their way at once
  for (int i0 = lo + lane; i0 < hi; i0 += 32 * U) {
    uint32_t key[U];
#pragma unroll
    for (int u = 0; u < U; ++u) key[u] = i0 + u * 32 < hi ? entry(i0 + u * 32).x : 0u;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * 32 < hi) atomicAdd(&cnt[warp * S + ((key[u] >> shift) & (bins - 1))], 1);
  }
  int all = 0, before = 0;
  const bool given = others(tid, all, before);      // (bins are at most half the threads)
  __syncthreads();
  if (tid < bins) {                                 // the warps' counts become how many tokens of the bin earlier warps have
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) {
      const int n = cnt[w * S + tid];
      cnt[w * S + tid] = run;
      run += n;
    }
    if (!given) all = run;
  }
  int up = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += v;
  }
  if (lane == 31) sums[warp] = up;
  __syncthreads();
  if (tid < bins) {
    int base = 0;
    for (int w = 0; w < warp; ++w) base += sums[w];
    place[tid] = base + up - all + before;
  }
  __syncthreads();
  for (int i0 = lo; i0 < hi; i0 += 32 * U) {
    uint2 e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) e[u] = i0 + u * 32 + lane < hi ? entry(i0 + u * 32 + lane) : make_uint2(0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * 32 >= hi) break;
      const int b = i0 + u * 32 + lane < hi ? static_cast<int>((e[u].x >> shift) & (bins - 1)) : -1;
      const uint32_t same = __match_any_sync(0xffffffffu, b);
      const int rank = __popc(same & ((1u << lane) - 1u));
      const int at = b >= 0 ? place[b] + cnt[warp * S + b] + rank : 0;
      __syncwarp();
      if (b >= 0 && rank == 0) cnt[warp * S + b] += __popc(same);
      __syncwarp();
      if (b >= 0) put(at, e[u]);
    }
  }
}

template <class From>
__global__ void __launch_bounds__(kThreads)
sort_rank_kernel(From from, SortArgs a, const int* __restrict__ hist, int chunks, uint2* __restrict__ out, Zero z) {
  pdl_wait();
  pdl_launch_dependents();
  if (static_cast<int>(blockIdx.x) >= z.from) return fill_zero(z);
  extern __shared__ int sm[];
  const int lo = blockIdx.x * a.chunk;
  sort_pass(min(a.T - lo, a.chunk), a.shift, a.bins, sm, [&](int i) { return from(lo + i, a); },
            [&](int bin, int& all, int& before) {
              if (bin < a.bins) {
#pragma unroll 16
                for (int c = 0; c < chunks; ++c) {
                  const int v = hist[static_cast<int64_t>(c) * a.bins + bin];
                  all += v;
                  before += c < static_cast<int>(blockIdx.x) ? v : 0;
                }
              }
              return true;
            },
            [&](int at, uint2 e) { out[at] = e; });
}

// The whole sort in one CTA while the others fill the gradient with zeros, the lists between its passes in shared memory up to kSharedSort tokens and in
// scratch memory above.
constexpr int kSharedSort = 8192;
template <class From>
__global__ void __launch_bounds__(kThreads)
sort_whole_kernel(From from, SortArgs a, int passes, uint2* __restrict__ out, uint2* __restrict__ other, Zero z) {
  pdl_wait();
  pdl_launch_dependents();
  if (static_cast<int>(blockIdx.x) >= z.from) return fill_zero(z);
  extern __shared__ int sm[];
  const int bits = 31 - __clz(a.bins);
  const bool shared = a.T <= kSharedSort;
  int* counts = sm + (shared ? 4 * a.T : 0);
  uint2* lists[2] = {shared ? reinterpret_cast<uint2*>(sm) : (passes & 1) ? out : other,      // (the last pass of an even number writes to `out`)
                     shared ? reinterpret_cast<uint2*>(sm) + a.T : (passes & 1) ? other : out};
  const auto own = [](int, int&, int&) { return false; };
  for (int p = 0; p < passes; ++p) {
    const uint2* in = lists[(p + 1) & 1];
    uint2* to = p + 1 == passes ? out : lists[p & 1];
    const auto write = [&](int at, uint2 e) { to[at] = e; };
    if (p == 0) sort_pass(a.T, 0, a.bins, counts, [&](int i) { return from(i, a); }, own, write);
    else sort_pass(a.T, p * bits, a.bins, counts, [&](int i) { return in[i]; }, own, write);
    __syncthreads();
  }
}

// ---- sums ---------------------------------------------------------------------------------------------
struct SumArgs {
  const uint2* sorted;       // (id, token), ids rising
  int T, chunk, V, D;
  int64_t ld;
  float scale;
  int* spans;                // how many runs go on behind the chunk that they begin in, and those chunks, in no order
  float* parts;              // [2 chunks][D]: what a chunk adds to the run that came in, and what it begins of the one that goes on
};

// A thread's four columns: next to each other (kFours), a CTA's width apart (kOnes), or two pairs that far apart (kPairs), which bf16 rows of an odd
// width or stride are read in, as 32-bit words, put together from two neighbouring ones where a row lies one column off them.
enum ColsBy { kFours, kOnes, kPairs };
template <ColsBy BY>
__device__ __forceinline__ int first_col(int step) {
  return blockIdx.y * step * 4 + threadIdx.x * (BY == kFours ? 4 : BY == kPairs ? 2 : 1);
}
template <ColsBy BY>
__device__ __forceinline__ int col_of(int col, int step, int j) {
  return BY == kFours ? col + j : BY == kOnes ? col + j * step : col + (j >> 1) * 2 * step + (j & 1);
}

// What a thread reads of a row, as it lies in memory (a conversion next to the load would wait for it).  at: its columns, those that are not there
// brought to 0 (they are not stored).  last: the row is the matrix' last one, behind which nothing is read (kPairs: of rows of two columns or more).
template <ColsBy BY, class T>
struct Cols;
template <>
struct Cols<kFours, float> {
  float4 x;
  __device__ __forceinline__ void load(const float* row, const int (&at)[4], bool) { x = *reinterpret_cast<const float4*>(row + at[0]); }
  __device__ __forceinline__ void add(float (&acc)[4]) const { acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w; }
};
template <>
struct Cols<kFours, __nv_bfloat16> {
  uint2 x;
  __device__ __forceinline__ void load(const __nv_bfloat16* row, const int (&at)[4], bool) { x = *reinterpret_cast<const uint2*>(row + at[0]); }
  __device__ __forceinline__ void add(float (&acc)[4]) const {
    acc[0] += __uint_as_float(x.x << 16);
    acc[1] += __uint_as_float(x.x & 0xffff0000u);
    acc[2] += __uint_as_float(x.y << 16);
    acc[3] += __uint_as_float(x.y & 0xffff0000u);
  }
};
template <class T>
struct Cols<kOnes, T> {
  T x[4];
  __device__ __forceinline__ void load(const T* row, const int (&at)[4], bool) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = row[at[j]];
  }
  __device__ __forceinline__ void add(float (&acc)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += to_f(x[j]);
  }
};
template <>
struct Cols<kPairs, __nv_bfloat16> {
  uint32_t x[2][2];
  bool off;
  __device__ __forceinline__ void load(const __nv_bfloat16* row, const int (&at)[4], bool last) {
    off = (reinterpret_cast<uintptr_t>(row) & 2) != 0;      // (columns of pairs are even)
    const char* words = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(row) & ~static_cast<uintptr_t>(3));
    if (!last) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[h][0] = *reinterpret_cast<const uint32_t*>(words + at[2 * h] * 2);
        x[h][1] = off ? *reinterpret_cast<const uint32_t*>(words + at[2 * h] * 2 + 4) : 0u;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {      // (at[2 h + 1] is the pair's second column, or 0)
        const uint32_t w = *reinterpret_cast<const uint16_t*>(row + at[2 * h]) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + at[2 * h + 1])) << 16;
        x[h][0] = off ? w << 16 : w;
        x[h][1] = w >> 16;
      }
    }
  }
  __device__ __forceinline__ void add(float (&acc)[4]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w = off ? __funnelshift_r(x[h][0], x[h][1], 16) : x[h][0];
      acc[2 * h] += __uint_as_float(w << 16);
      acc[2 * h + 1] += __uint_as_float(w & 0xffff0000u);
    }
  }
};

template <ColsBy BY, class T>
__device__ __forceinline__ void store_cols(T* row, int col, int step, int D, const float (&x)[4]) {
  if constexpr (BY == kFours) {
    store4(row + col, x);
  } else {
    T* first = row + col;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = col_of<BY>(0, step, j);
      if (col + c < D) put(first + c, x[j]);
    }
  }
}

template <class S, class O, ColsBy BY, int STEP>
__global__ void __launch_bounds__(STEP)
segment_sum_kernel(SumArgs a, const S* __restrict__ dout, O* __restrict__ dtable) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int step = STEP;
  const int col = first_col<BY>(step);
  const int lo = blockIdx.x * a.chunk, hi = min(a.T, lo + a.chunk);
  if (col >= a.D) return;
  int at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) at[j] = col_of<BY>(col, step, j) < a.D ? col_of<BY>(col, step, j) : 0;
  const uint32_t none = static_cast<uint32_t>(a.V);
  const uint32_t came = lo > 0 ? a.sorted[lo - 1].x : none, goes = hi < a.T ? a.sorted[hi].x : none;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t run = a.sorted[lo].x;
  bool open = run == came;           // the run began before this chunk
  // a run that begins here and goes on is one for the next kernel
  if (threadIdx.x == 0 && blockIdx.y == 0 && goes != none && a.sorted[hi - 1].x == goes && came != goes) a.spans[1 + atomicAdd(a.spans, 1)] = blockIdx.x;
  if (run == none) return;
  constexpr int U = 8;
  static_assert(kSegMin % U == 0, "chunks of whole steps");
  uint2 next[U];                     // entries behind the end: no row, and the first token's to read
  const auto fetch = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = i0 + u < hi ? a.sorted[i0 + u] : make_uint2(none, 0);
  };
  fetch(lo);
  for (int i0 = lo; i0 < hi; i0 += U) {
    uint32_t id[U];
    Cols<BY, S> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      id[u] = next[u].x;
      x[u].load(dout + static_cast<int64_t>(next[u].y) * a.ld, at, static_cast<int>(next[u].y) + 1 == a.T);
    }
    fetch(i0 + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (id[u] != run) {
        if (open) {
          store_cols<BY>(a.parts + static_cast<int64_t>(2 * blockIdx.x) * a.D, col, step, a.D, acc);
        } else if (!(i0 + u >= hi && run == goes)) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] *= a.scale;
          store_cols<BY>(dtable + static_cast<int64_t>(run) * a.D, col, step, a.D, acc);
        } else {
          store_cols<BY>(a.parts + static_cast<int64_t>(2 * blockIdx.x + 1) * a.D, col, step, a.D, acc);
        }
        if (id[u] == none) return;
        run = id[u];
        open = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = 0.f;
      }
      x[u].add(acc);
    }
  }
  // a chunk of whole steps: its last run
  if (open) {
    store_cols<BY>(a.parts + static_cast<int64_t>(2 * blockIdx.x) * a.D, col, step, a.D, acc);
  } else if (run == goes) {
    store_cols<BY>(a.parts + static_cast<int64_t>(2 * blockIdx.x + 1) * a.D, col, step, a.D, acc);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] *= a.scale;
    store_cols<BY>(dtable + static_cast<int64_t>(run) * a.D, col, step, a.D, acc);
  }
}

// Runs over several chunks: what a run left in the chunk that it begins in, and in those up to its end
template <class O>
__global__ void __launch_bounds__(kSegThreads)
segment_join_kernel(SumArgs a, O* __restrict__ dtable) {
  pdl_wait();
  pdl_launch_dependents();
  const int tiles = (a.D + kJoinCols - 1) / kJoinCols, items = a.spans[0] * tiles;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int c = a.spans[1 + item / tiles], tile = item % tiles;
    const uint32_t run = a.sorted[(c + 1) * a.chunk].x;
    // its last chunk: the first one behind this whose last token is another's (all chunks that could be are asked at once)
    __shared__ int ends;
    __syncthreads();
    if (threadIdx.x == 0) ends = 0x7fffffff;
    __syncthreads();
    for (int i0 = c + 1; ends == 0x7fffffff; i0 += kSegThreads) {
      const int i = i0 + threadIdx.x;
      const int64_t behind = (static_cast<int64_t>(i) + 1) * a.chunk;
      const bool over = behind >= a.T || a.sorted[behind - 1].x != run || a.sorted[behind].x != run;
      __syncthreads();
      if (over) atomicMin(&ends, i);
      __syncthreads();
    }
    const int end = ends;
    // a warp adds up every eighth part, four columns a thread
    constexpr int kTeams = kSegThreads / 32;
    __shared__ float sums[kTeams][kJoinCols];
    const int team = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int i = c + team; i <= end; i += kTeams) {
      const float* part = a.parts + static_cast<int64_t>(2 * i + (i == c ? 1 : 0)) * a.D;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = tile * kJoinCols + lane + j * 32;
        acc[j] += part[col < a.D ? col : 0];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[team][lane + j * 32] = acc[j];
    __syncthreads();
    const int n = threadIdx.x, col = tile * kJoinCols + n;
    if (n < kJoinCols && col < a.D) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kTeams; ++w) s += sums[w][n];
      put(dtable + static_cast<int64_t>(run) * a.D + col, s * a.scale);
    }
  }
}

int bits_of(int64_t n) {             // of the largest value below n
  int b = 1;
  while ((1ll << b) < n) ++b;
  return b;
}
// One CTA sorts what fits its shared memory, and up to twice that where the zeros take longer than it does: 16384 tokens over 102 MB of bf16
// rows 80 us so and 66 by many CTAs in four kernels, over 311 MB 90 and 100, over 622 MB of fp32 rows 185 and 194; 32768 over 622 MB 274 and 271.
bool sorts_whole(int64_t T, int64_t bytes) { return T <= kSharedSort || (T <= 2 * kSharedSort && bytes >= 18000 * T); }

struct Plan {
  bool whole;                        // sorted by one CTA
  int passes, bits, chunks, chunk, seg_chunk, seg_chunks;
};
Plan plan_for(int64_t T, int64_t V, int64_t bytes) {
  Plan p{};
  const int bits = bits_of(V + 1);
  p.passes = (bits + kDigit - 1) / kDigit;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.whole = sorts_whole(T, bytes);
  p.chunk = static_cast<int>((T + kMaxChunks - 1) / kMaxChunks);
  p.chunk = p.whole ? static_cast<int>(T) : p.chunk < 2 * kThreads ? 2 * kThreads : (p.chunk + kThreads - 1) / kThreads * kThreads;
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
  const int warps = T < 8 ? static_cast<int>(T) : 8, slices = (D + kRowCols - 1) / kRowCols;
  int64_t rows = (T + warps - 1) / warps;
  const int64_t most = (148 * 8 + slices - 1) / slices;
  const dim3 block(32 * warps), grid(static_cast<unsigned>(rows < most ? rows : most), slices);
  const auto run = [&](auto* kernel) { return launch_code(launch_pdl(kernel, grid, block, 0, stream, ids, table, ld, out, scale, T, V, D)); };
  if (vec) return run(embedding_rows_kernel<I, S, O, kRowsFours>);
  if constexpr (sizeof(S) == 2 && sizeof(O) == 2) {
    if (aligned(table, 4) && aligned(out, 4) && ld >= D) return run(embedding_rows_kernel<I, S, O, kRowsPairs>);
  }
  return run(embedding_rows_kernel<I, S, O, kRowsOnes>);
}

template <class S, class O>
int launch_sums(const SumArgs& a, int chunks, const S* dout, O* dtable, cudaStream_t stream) {
  const bool vec = a.D % 4 == 0 && a.ld % 4 == 0 && aligned(dout, 4 * sizeof(S)) && aligned(dtable, 4 * sizeof(O));
  const auto run = [&](auto* kernel, int width) {
    return launch_code(launch_pdl(kernel, dim3(chunks, (a.D + width * 4 - 1) / (width * 4)), dim3(width), 0, stream, a, dout, dtable));
  };
  constexpr ColsBy kWords = sizeof(S) == 2 ? kPairs : kOnes;
  // A pair's second word ends at most two columns behind its row's last: in the next row, unless rows are one value each (of an odd number the last
  // but one would read behind the matrix).
  const bool words = sizeof(S) == 2 && aligned(dout, 4) && a.ld >= a.D && a.D > 1, wide = a.D > 256;      // narrow rows take CTAs of two warps
  int rc;
  if (vec) rc = wide ? run(segment_sum_kernel<S, O, kFours, kSegThreads>, kSegThreads) : run(segment_sum_kernel<S, O, kFours, 64>, 64);
  else if (words) rc = wide ? run(segment_sum_kernel<S, O, kWords, kSegThreads>, kSegThreads) : run(segment_sum_kernel<S, O, kWords, 64>, 64);
  else rc = wide ? run(segment_sum_kernel<S, O, kOnes, kSegThreads>, kSegThreads) : run(segment_sum_kernel<S, O, kOnes, 64>, 64);
  if (rc == 0 && chunks > 1) {
    const int64_t items = static_cast<int64_t>(chunks - 1) * ((a.D + kJoinCols - 1) / kJoinCols);
    rc = launch_code(launch_pdl(segment_join_kernel<O>, dim3(static_cast<unsigned>(items < 148 * 8 ? items : 148 * 8)), dim3(kSegThreads), 0, stream,
                                a, dtable));
  }
  return rc;
}

bool fits(int64_t T, int64_t V, int D) {
  return T >= 1 && T <= (1ll << 30) && V >= 1 && V <= (1ll << 30) && D >= 1 && D <= (1 << 16);
}

}  // namespace

int64_t embedding_scratch_bytes(int64_t T, int64_t V, int D, bool dtable16) {
  const Plan p = plan_for(T, V, V * D * (dtable16 ? 2 : 4));
  return 2 * on16(8 * T) + on16(4ll * p.chunks << p.bits) + on16(4ll * (p.seg_chunks + 1)) + 8ll * p.seg_chunks * D;
}

int embedding_grad_kernels(int64_t T, int64_t V, int D, bool dtable16) {
  const Plan p = plan_for(T, V, V * D * (dtable16 ? 2 : 4));
  return (p.whole ? 1 : 2 * p.passes) + (p.seg_chunks > 1 ? 2 : 1);
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
  const int64_t bytes = V * D * (dtable16 ? 2 : 4);
  const Plan p = plan_for(T, V, bytes);
  char* at = static_cast<char*>(scratch);
  uint2* lists[2] = {reinterpret_cast<uint2*>(at), reinterpret_cast<uint2*>(at + on16(8 * T))};
  at += 2 * on16(8 * T);
  int* hist = reinterpret_cast<int*>(at);
  at += on16(4ll * p.chunks << p.bits);
  int* spans = reinterpret_cast<int*>(at);
  at += on16(4ll * (p.seg_chunks + 1));
  SortArgs a{};
  a.T = static_cast<int>(T); a.chunk = p.chunk; a.bins = 1 << p.bits; a.V = static_cast<int>(V); a.padding = static_cast<int>(padding);
  // the kernels that rank tokens fill the gradient, each its share (those that count are done before a share would be)
  const int kernels = p.whole ? 1 : p.passes;
  int64_t done = 0;
  Zero z{static_cast<char*>(dtable), 0, 0, p.chunks, spans};
  const auto share = [&](int i) {
    z.lo = done;
    z.hi = done = i + 1 == kernels ? bytes : bytes * (i + 1) / kernels / 16 * 16;
    // 256 KB for each, so that SMs which are done take more (147 CTAs that share it out: 105 us for 622 MB, so 89), 64 KB where that leaves SMs idle
    const int64_t n = z.hi - z.lo, idle = (n + (1 << 16) - 1) >> 16, many = (n + (1 << 18) - 1) >> 18;
    const int64_t ctas = idle < 147 ? idle : many < 147 ? 147 : many;
    return static_cast<int>(ctas < 1 ? 1 : ctas);
  };
  const int smem = 4 * rank_ints(a.bins) + (p.whole && T <= kSharedSort ? 16 * a.T : 0);
  const auto whole = [&](auto from) {
    using From = decltype(from);
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(sort_whole_kernel<From>), smem)) return -20;
    const int more = share(0);
    return launch_code(launch_pdl(sort_whole_kernel<From>, dim3(1 + more), dim3(kThreads), static_cast<size_t>(smem), stream, from, a, p.passes,
                                  lists[0], lists[1], z));
  };
  const auto pass = [&](auto from, int i) {
    using From = decltype(from);
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(sort_rank_kernel<From>), smem)) return -20;
    a.shift = i * p.bits;
    const int rc = launch_code(launch_pdl(sort_count_kernel<From>, dim3(p.chunks), dim3(kThreads), 0, stream, from, a, hist));
    if (rc) return rc;
    const int more = share(i);
    return launch_code(launch_pdl(sort_rank_kernel<From>, dim3(p.chunks + more), dim3(kThreads), static_cast<size_t>(smem), stream, from, a,
                                  hist, p.chunks, lists[i & 1], z));
  };
  if (p.whole) {
    const int rc = ids64 ? whole(FromIds64{static_cast<const int64_t*>(ids)}) : whole(FromIds32{static_cast<const int*>(ids)});
    if (rc) return rc;
  }
  for (int i = 0; i < p.passes && !p.whole; ++i) {
    const int rc = i > 0 ? pass(FromPass{lists[(i - 1) & 1]}, i)
                   : ids64 ? pass(FromIds64{static_cast<const int64_t*>(ids)}, i)
                           : pass(FromIds32{static_cast<const int*>(ids)}, i);
    if (rc) return rc;
  }
  SumArgs s{};
  s.sorted = lists[p.whole ? 0 : (p.passes - 1) & 1];
  s.T = a.T; s.chunk = p.seg_chunk; s.V = a.V; s.D = D; s.ld = ld; s.scale = scale;
  s.spans = spans;
  s.parts = reinterpret_cast<float*>(at);
  const auto sums = [&](auto* d) {
    return dtable16 ? launch_sums(s, p.seg_chunks, d, static_cast<__nv_bfloat16*>(dtable), stream)
                    : launch_sums(s, p.seg_chunks, d, static_cast<float*>(dtable), stream);
  };
  return dout16 ? sums(static_cast<const __nv_bfloat16*>(dout)) : sums(static_cast<const float*>(dout));
}

}  // namespace tb
