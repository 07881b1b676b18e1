// AdamW over many tensors whose two moments are held in 8 bits, one launch, and the moments read back.
//
// A block of 128 consecutive values of a tensor has one fp32 scale.  With a the block's largest magnitude, a magnitude x is brought to
// y = x TOP / a + FIRST and held as y's fp32 pattern cut to 3 bits of mantissa, counted from FIRST's pattern:
//   code = ((bits(y) + (r << 4)) >> 20) - (bits(FIRST) >> 20),   x kept = (value(code) - FIRST) a / TOP
// (even steps next to zero, steps of an eighth further up).  First moment: a sign bit and FIRST = 2^-15, 127 steps down to a 2^-19; second
// moment: FIRST = 2^-31, 255 steps down to a 2^-35.  Either is off by a step of its code at most, (|x| + FIRST a / TOP) / 8: an eighth of large
// values, half of a first moment at a 2^-18.  r are 16 random bits: a value goes to one of its two neighbours with the probability that makes the
// mean its own.  To the nearest, a second moment that changes by 1 - beta2 of
// itself a step, less than half a step of the code, would stay where it is for good.  A second moment above zero keeps at least the first step:
// no update divides by eps alone where the gradients have been small beside the block's.  That step's root is a 2^-17.45 of the second moments' a:
// elements with gradients down to 2^-17.45 of the block's largest move as in 32 bits, those below are damped in proportion (0.69 of the way
// at 2^-18, 0.38 at 2^-18.9).
// A block that holds something that is not finite reads back as NaN, one whose largest magnitude is under 2^-100 as zeros.
//
// Random bits: h(i) = mix(key ^ low 32 bits of i), key from (seed, step, the tensor's number, high bits of i), mix two rounds of xorshift and multiplication
// (constants by C. Wellons, 2018); 16 bits for each moment.
//
// The moments' arithmetic is fp32, every operation rounded by itself in the order written (no contraction): their codes are those of the same
// statements in plain tensor operations, bit for bit.
//
// Bound by memory: an element reads 4 + 4 + 1 + 1 bytes and writes 4 + 1 + 1 (+ 2 of the bf16 shadow), 18.1 with the scales, against 30 with the
// moments in fp32.  64 Mi elements with the shadow 208 us (5.9 TB/s; a plain copy has 6.55), 73 instructions an element and issue slots 69 % taken;
// 275 M in 17 tensors 817 us, 760 at copy bandwidth.  A moment read back as bf16: 275 M values in 127 us, 126 at copy bandwidth; 64 Mi in 36.
#include "api.h"
#include "common.cuh"

namespace tb {

namespace {

constexpr int kThreads = 256;
constexpr int kSmallChunk = kChunkElems / 4;      // where there are too few chunks of kChunkElems for the SMs
constexpr float kFirstM = 3.0517578125e-05f, kFirstV = 4.656612873077393e-10f;      // 2^-15, 2^-31
constexpr uint32_t kKeyM = 896, kKeyV = 768;                                            // their patterns >> 20
constexpr float kTopM = 1.875f - 3.0517578125e-05f, kTopV = 1.875f;
constexpr float kTinyBlock = 7.888609052210118e-31f;      // 2^-100

constexpr uint32_t kMix1 = 0x7feb352du, kMix2 = 0x846ca68bu;
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * kMix1;
  x = (x ^ (x >> 15)) * kMix2;
  return x ^ (x >> 16);
}

// Value J of four codes, over its sign.  (A code in bits 20 and up does not meet the bits of its KEY.)
template <bool SIGNED, int J>
__device__ __forceinline__ float decode8(uint32_t codes, float scale) {
  const uint32_t at20 = J < 3 ? codes << (20 - 8 * J) : codes >> 4;
  const float y = __uint_as_float((at20 & (SIGNED ? 0x07f00000u : 0x0ff00000u)) | ((SIGNED ? kKeyM : kKeyV) << 20));
  // (a first moment's y - FIRST and FIRST scale are exact: one rounding either way)
  if (SIGNED) return __uint_as_float(__float_as_uint(fmaf(y, scale, -kFirstM * scale)) ^ ((codes << (24 - 8 * J)) & 0x80000000u));
  return __fmul_rn(y - kFirstV, scale);
}

// What a block is rounded with.  Half of a warp works it out for the first moment, half for the second.
struct Coder {
  float scale;             // of this half's moment
  float m, v;              // both inverses, negative for a block of zeros or NaN
};
__device__ __forceinline__ Coder coder_for(uint32_t m_top, uint32_t v_top) {
  const bool first = (threadIdx.x & 16) == 0;
  const float top = __uint_as_float(first ? m_top : v_top), most = first ? kTopM : kTopV;
  const float over = first ? static_cast<float>(1.0 / static_cast<double>(kTopM)) : static_cast<float>(1.0 / static_cast<double>(kTopV));
  const bool fine = top >= kTinyBlock && top < INFINITY;
  const float inverse = fine ? __fmul_rn(__frcp_rn(top), most) : -1.f;
  Coder c;
  c.scale = fine ? __fmul_rn(top, over) : top < kTinyBlock ? 0.f : __uint_as_float(0x7fc00000u);
  c.m = __shfl_sync(0xffffffffu, inverse, 0);
  c.v = __shfl_sync(0xffffffffu, inverse, 16);
  return c;
}
// The pattern of |x| brought to the block's range, plus 16 random bits below those that are kept, four bits up: the code is the highest byte (of
// a first moment its lower 7 bits).  y is at most a few units above 1.875, the random bits at most 16 units short of a step: the largest code is
// not passed.  r: the random bits in bytes 1 and 2.
template <bool SIGNED>
__device__ __forceinline__ uint32_t round8(float x, float inverse, uint32_t r) {
  return __float_as_uint(__fadd_rn(__fmul_rn(fabsf(x), inverse), SIGNED ? kFirstM : kFirstV)) * 16u + r;
}
__device__ __forceinline__ uint32_t high_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073u), __byte_perm(c, d, 0x0073u), 0x5410u);
}

// f(0), f(1), f(2), f(3) with the number as a type
template <int J>
struct Num { static constexpr int value = J; };
template <class F>
__device__ __forceinline__ void four(F f) {
  f(Num<0>{});
  f(Num<1>{});
  f(Num<2>{});
  f(Num<3>{});
}

// Four consecutive values of which `left` are there
__device__ __forceinline__ void load4(const float* p, bool vec, int left, float (&x)[4]) {
  if (vec && left >= 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = j < left ? p[j] : 0.f;
  }
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, bool vec, int left, float (&x)[4]) {
  if (vec && left >= 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = j < left ? __bfloat162float(p[j]) : 0.f;
  }
}
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, bool vec, int left) {
  if (vec && left >= 4) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) c |= j < left ? static_cast<uint32_t>(p[j]) << (8 * j) : 0u;
  return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, bool vec, int left, uint32_t c) {
  if (vec && left >= 4) {
    *reinterpret_cast<uint32_t*>(p) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = static_cast<uint8_t>(c >> (8 * j));
  }
}
__device__ __forceinline__ void store4(float* p, bool vec, int left, const float (&x)[4]) {
  if (vec && left >= 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = x[j];
  }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, bool vec, int left, const float (&x)[4]) {
  if (vec && left >= 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = __float2bfloat16(x[j]);
  }
}
__device__ __forceinline__ bool on(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Root and quotient of the update are the approximate instructions (2 units each): what they cost otherwise, half of all instructions, made the
// kernel 1.6 times slower.  They touch the parameters only, by 2^-21 of an update; the moments keep the bits of the plain statement.
__device__ __forceinline__ float update(float p, float m, float v, const Adam8Scalars& s) {
  float root, over;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(root) : "f"(v), "f"(1.17549435e-38f));      // (not zero: also with eps 0 no 0 / 0; a NaN stays one)
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(root));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(over) : "f"(fmaf(root, s.root, s.eps)));
  return fmaf(-s.step_size, m * over, p * s.decay);
}

// The addresses of up to kState8ByValue tensors as an argument of the kernel: new gradients, at new addresses every step, then cost no copy to the
// device (30 us of the host's time for a pinned one).  COLUMNS 0: they lie on the device.
template <int COLUMNS>
struct Addresses {
  int64_t p[COLUMNS * kState8ByValue];
};
template <>
struct Addresses<0> {};
template <int COLUMNS>
__device__ __forceinline__ int64_t address(const State8List& t, const Addresses<COLUMNS>& a, int column, int ti) {
  if constexpr (COLUMNS == 0) return t.ptrs[column * t.n_tensors + ti];
  else return a.p[column * t.n_tensors + ti];
}

struct Four {
  float p[4], g[4];
  uint32_t m, v;           // codes
  float ms, vs;            // scales
  float scale;             // afterwards: lanes 0 to 15 the first moment's, the others the second's
};

// One thread's four values of a warp's block, element i the first of them
__device__ __forceinline__ void step4(Four& f, const Adam8Scalars& s, float gs, uint32_t key, uint32_t i) {
  float mx[4], vx[4];
  uint32_t m_top = 0, v_top = 0;
  four([&](auto num) {
    constexpr int j = decltype(num)::value;
    const float g = __fmul_rn(f.g[j], gs);
    mx[j] = __fadd_rn(__fmul_rn(decode8<true, j>(f.m, f.ms), s.beta1), __fmul_rn(g, s.rest1));
    vx[j] = __fadd_rn(__fmul_rn(decode8<false, j>(f.v, f.vs), s.beta2), __fmul_rn(__fmul_rn(g, s.rest2), g));
    f.p[j] = update(f.p[j], mx[j], vx[j], s);
    // (patterns of magnitudes are ordered as they are, NaN last)
    m_top = max(m_top, __float_as_uint(fabsf(mx[j])));
    v_top = max(v_top, __float_as_uint(fabsf(vx[j])));
  });
  const Coder c = coder_for(__reduce_max_sync(0xffffffffu, m_top), __reduce_max_sync(0xffffffffu, v_top));
  uint32_t mo[4], vo[4];
  // mix32(key ^ (i + j)) for an i that is a multiple of 4: its first step is the same for all but the last bits
  const uint32_t x0 = key ^ i, mixed = x0 ^ (x0 >> 16);
  four([&](auto num) {
    constexpr int j = decltype(num)::value;
    uint32_t h = (mixed ^ j) * kMix1;
    h = (h ^ (h >> 15)) * kMix2;
    mo[j] = round8<true>(mx[j], c.m, __byte_perm(h ^ (h >> 16), 0u, 0x4104u));
    vo[j] = round8<false>(vx[j], c.v, __byte_perm(h, 0u, 0x4324u));
  });
  if (min(min(vo[0], vo[1]), min(vo[2], vo[3])) < 1u << 24) {      // a second moment above zero keeps the first step
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (vx[j] > 0.f) vo[j] = max(vo[j], 1u << 24);
  }
  const uint32_t sign = high_bytes(__float_as_uint(mx[0]), __float_as_uint(mx[1]), __float_as_uint(mx[2]), __float_as_uint(mx[3]));
  const uint32_t m = high_bytes(mo[0], mo[1], mo[2], mo[3]), v = high_bytes(vo[0], vo[1], vo[2], vo[3]);
  f.m = c.m > 0.f ? (m & 0x7f7f7f7fu) | (sign & 0x80808080u) : 0u;
  f.v = c.v > 0.f ? v : 0u;
  f.scale = c.scale;
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(BYTES) : "memory");
}
constexpr int kStages = 4;
struct Stage {               // a warp's block
  float4 g[32];
  uint32_t codes[2][32];     // first moment, second moment
  float scales[2];
  float unused[2];
};

struct Chunk {               // where a chunk's tensors begin
  float* p;
  const char* g;
  uint8_t *m, *v;
  float *m_scale, *v_scale;
  __nv_bfloat16* sh;
};

// A chunk of whole rounds on 16-byte boundaries, a warp per block of 128, four values a thread.  The values of the next three rounds are on their
// way to shared memory meanwhile: held in registers they would leave room for too few warps, and without them the loads of a round wait
// behind the stores of the one before, which for all the compiler knows could be to the same place.
template <bool G16, bool SHADOW>
__device__ __forceinline__ void whole_chunk(const Chunk& c, int count, const Adam8Scalars& s, float gs, uint32_t key, uint32_t i0, Stage* stages) {
  constexpr int kStep = kThreads / 32 * kStateBlock, kAhead = kStages - 1;
  static_assert(kSmallChunk % (kStages * kStep) == 0 && kChunkElems % kSmallChunk == 0, "whole rounds");
  const int lane = threadIdx.x & 31, first = (threadIdx.x >> 5) * kStateBlock, at = first + lane * 4;
  // each thread's places, moved on by kStages rounds at a time
  float* p = c.p + at;
  const char* g = c.g + at * (G16 ? 2 : 4);
  uint8_t *m = c.m + at, *v = c.v + at;
  __nv_bfloat16* sh = c.sh + at;
  float* scale = (lane < 16 ? c.m_scale : c.v_scale) + first / kStateBlock;
  // lanes 0 to 7 copy the first moment's codes, 16 to 23 the second's, 8 and 24 the scales
  const uint8_t* codes = (lane < 16 ? c.m : c.v) + first + (lane & 7) * 16;
  const bool copies_codes = (lane & 8) == 0, copies_scale = (lane & 15) == 8;
  const auto fetch = [&](int r, Stage& st) {
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p + r * kStep));      // (staged with the rest it is 20 us slower, of 208)
    copy_async<G16 ? 8 : 16>(&st.g[lane], g + r * kStep * (G16 ? 2 : 4));
    if (copies_codes) copy_async<16>(&st.codes[lane >> 4][(lane & 7) * 4], codes + r * kStep);
    if (copies_scale) copy_async<4>(&st.scales[lane >> 4], scale + r * (kStep / kStateBlock));
  };
#pragma unroll
  for (int r = 0; r < kAhead; ++r) {
    fetch(r, stages[r]);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  uint32_t i = i0 + at;
#pragma unroll 1
  for (int left = count / kStep; left > 0; left -= kStages) {
#pragma unroll
    for (int r = 0; r < kStages; ++r) {
      // (the stage that is filled here was read by all lanes in the round before)
      if (r == 0 || left > kStages) fetch(r + kAhead, stages[(r + kAhead) % kStages]);
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
      __syncwarp();
      const Stage& st = stages[r];
      Four f;
      load4(p + r * kStep, true, 4, f.p);      // (needed last of all, and in L2 by now)
      if (G16) load4(reinterpret_cast<const __nv_bfloat16*>(&st.g[lane]), true, 4, f.g);
      else load4(reinterpret_cast<const float*>(&st.g[lane]), true, 4, f.g);
      f.m = st.codes[0][lane];
      f.v = st.codes[1][lane];
      f.ms = st.scales[0];
      f.vs = st.scales[1];
      __syncwarp();
      step4(f, s, gs, key, i + r * kStep);
      store4(p + r * kStep, true, 4, f.p);
      if (SHADOW) store4(sh + r * kStep, true, 4, f.p);
      store_codes(m + r * kStep, true, 4, f.m);
      store_codes(v + r * kStep, true, 4, f.v);
      if ((lane & 15) == 0) scale[r * (kStep / kStateBlock)] = f.scale;
    }
    p += kStages * kStep;
    g += kStages * kStep * (G16 ? 2 : 4);
    m += kStages * kStep;
    v += kStages * kStep;
    if (SHADOW) sh += kStages * kStep;
    codes += kStages * kStep;
    scale += kStages * (kStep / kStateBlock);
    i += kStages * kStep;
  }
}

template <int COLUMNS>
__global__ void __launch_bounds__(kThreads, 4)
adamw8_kernel(State8List t, Adam8Scalars s, const float* __restrict__ grad_scale, const float* __restrict__ hyper,
              const __grid_constant__ Addresses<COLUMNS> addresses) {
  pdl_wait();
  pdl_launch_dependents();
  uint32_t key = s.key;
  if (hyper) {      // what changes from step to step read from device memory: the launch can be replayed from a graph
    s.step_size = hyper[0];
    s.root = hyper[1];
    s.decay = hyper[2];
    key = __float_as_uint(hyper[3]);
  }
  const int ti = t.block_tensor[blockIdx.x];
  const int64_t n = t.numel[ti], lo = static_cast<int64_t>(t.block_chunk[blockIdx.x]) * t.chunk;
  const int count = static_cast<int>(lo + t.chunk < n ? t.chunk : n - lo);
  const auto ptr = [&](int column) { return address<COLUMNS>(t, addresses, column, ti); };
  float* p = reinterpret_cast<float*>(ptr(0)) + lo;
  const char* g = reinterpret_cast<const char*>(ptr(1));
  uint8_t* m = reinterpret_cast<uint8_t*>(ptr(2)) + lo;
  uint8_t* v = reinterpret_cast<uint8_t*>(ptr(3)) + lo;
  float* m_scale = reinterpret_cast<float*>(ptr(4)) + lo / kStateBlock;
  float* v_scale = reinterpret_cast<float*>(ptr(5)) + lo / kStateBlock;
  __nv_bfloat16* sh = reinterpret_cast<__nv_bfloat16*>(ptr(6));
  const int flags = t.flags[ti];
  const bool g16 = (flags & 1) != 0;
  g += lo * (g16 ? 2 : 4);
  if (sh) sh += lo;
  const bool vp = on(p, 16), vg = on(g, g16 ? 8 : 16), vm = on(m, 16), vv = on(v, 16), vs = on(sh, 8);
  float gs = grad_scale ? *grad_scale : 1.f;
  if (s.maximize) gs = -gs;
  key = mix32(key + 0x85ebca6bu * static_cast<uint32_t>(flags >> 1) + 0xc2b2ae35u * static_cast<uint32_t>(lo >> 32));
  const int lane = threadIdx.x & 31, first = (threadIdx.x >> 5) * kStateBlock;
  constexpr int kStep = kThreads / 32 * kStateBlock;
  if (count == t.chunk && vp && vg && vm && vv && vs) {
    extern __shared__ __align__(16) uint8_t dynamic[];      // [warps][kStages]
    Stage* stages = reinterpret_cast<Stage*>(dynamic);
    const Chunk c{p, g, m, v, m_scale, v_scale, sh};
    Stage* mine = stages + (threadIdx.x >> 5) * kStages;
    const uint32_t i0 = static_cast<uint32_t>(lo);
    if (g16) sh ? whole_chunk<true, true>(c, count, s, gs, key, i0, mine) : whole_chunk<true, false>(c, count, s, gs, key, i0, mine);
    else sh ? whole_chunk<false, true>(c, count, s, gs, key, i0, mine) : whole_chunk<false, false>(c, count, s, gs, key, i0, mine);
    return;
  }
  // a tensor's last chunk, or one that does not lie on 16 bytes: what is not there is read as zero, which is no block's largest
  for (int b = first; b < count; b += kStep) {
    const int i = b + lane * 4, left = max(0, min(4, count - i));
    Four f;
    load4(p + i, vp, left, f.p);
    if (g16) load4(reinterpret_cast<const __nv_bfloat16*>(g) + i, vg, left, f.g);
    else load4(reinterpret_cast<const float*>(g) + i, vg, left, f.g);
    f.m = load_codes(m + i, vm, left);
    f.v = load_codes(v + i, vv, left);
    f.ms = m_scale[b / kStateBlock];
    f.vs = v_scale[b / kStateBlock];
    // (a NaN scale is the block's, and no value of its own where there is none: code 0 times NaN)
    step4(f, s, gs, key, static_cast<uint32_t>(lo) + i);
    store4(p + i, vp, left, f.p);
    if (sh) store4(sh + i, vs, left, f.p);
    store_codes(m + i, vm, left, f.m);
    store_codes(v + i, vv, left, f.v);
    if ((lane & 15) == 0) (lane == 0 ? m_scale : v_scale)[b / kStateBlock] = f.scale;
  }
}

// ptrs: codes, scales, and the values' place in `all`, in elements
template <class T, bool SIGNED, int COLUMNS>
__global__ void __launch_bounds__(kThreads)
state8_values_kernel(State8List t, T* __restrict__ all, const __grid_constant__ Addresses<COLUMNS> addresses) {
  pdl_wait();
  pdl_launch_dependents();
  const int ti = t.block_tensor[blockIdx.x];
  const int64_t n = t.numel[ti], lo = static_cast<int64_t>(t.block_chunk[blockIdx.x]) * t.chunk;
  const int64_t hi = lo + t.chunk < n ? lo + t.chunk : n;
  const auto ptr = [&](int column) { return address<COLUMNS>(t, addresses, column, ti); };
  const uint8_t* codes = reinterpret_cast<const uint8_t*>(ptr(0));
  const float* scales = reinterpret_cast<const float*>(ptr(1));
  T* out = all + ptr(2);
  const bool vc = on(codes, 4), vo = on(out, 4 * sizeof(T));
  if (hi - lo == t.chunk && on(codes, 8) && on(out, 16)) {      // eight values a thread: whole lines in and out
    const int rounds = t.chunk / (kThreads * 8);
    const uint2* from = reinterpret_cast<const uint2*>(codes + lo) + threadIdx.x;
    const float* scale = scales + lo / kStateBlock + threadIdx.x / (kStateBlock / 8);
    T* to = out + lo + threadIdx.x * 8;
    const auto go = [&](auto flight) {      // so many rounds' loads on their way at once
      constexpr int kFlight = decltype(flight)::value;
      static_assert(kSmallChunk % (2 * kThreads * 8) == 0 && kChunkElems % (4 * kThreads * 8) == 0, "whole rounds");
#pragma unroll 1
    for (int r0 = 0; r0 < rounds; r0 += kFlight) {
      uint2 c[kFlight];
      float s[kFlight];
#pragma unroll
      for (int r = 0; r < kFlight; ++r) {
        c[r] = from[(r0 + r) * kThreads];
        s[r] = scale[(r0 + r) * (kThreads * 8 / kStateBlock)];
      }
#pragma unroll
      for (int r = 0; r < kFlight; ++r) {
        float x[4], y[4];
        four([&](auto num) {
          constexpr int j = decltype(num)::value;
          x[j] = decode8<SIGNED, j>(c[r].x, s[r]);
          y[j] = decode8<SIGNED, j>(c[r].y, s[r]);
        });
        T* at = to + (r0 + r) * (kThreads * 8);
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(at) =
              make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
        } else {
          store4(at, true, 4, x);
          store4(at + 4, true, 4, y);
        }
      }
    }
    };
    if (rounds % 4 == 0) go(Num<4>{});
    else go(Num<2>{});
    return;
  }
  for (int64_t i = lo + threadIdx.x * 4; i < hi; i += kThreads * 4) {
    const int left = static_cast<int>(hi - i < 4 ? hi - i : 4);
    const uint32_t c = load_codes(codes + i, vc, left);
    const float scale = scales[i / kStateBlock];
    float x[4];
    four([&](auto num) {
      constexpr int j = decltype(num)::value;
      x[j] = decode8<SIGNED, j>(c, scale);
    });
    store4(out + i, vo, left, x);
  }
}

template <int COLUMNS>
Addresses<COLUMNS> addresses_of(const State8List& t) {
  Addresses<COLUMNS> a{};
  if constexpr (COLUMNS > 0)
    for (int i = 0; i < COLUMNS * t.n_tensors; ++i) a.p[i] = t.host_ptrs[i];
  return a;
}

bool fits(const State8List& t) {
  return (t.chunk == kChunkElems || t.chunk == kSmallChunk) && (t.host_ptrs == nullptr || t.n_tensors <= kState8ByValue);
}

template <int COLUMNS>
int launch_step(const State8List& t, const Adam8Scalars& s, const float* grad_scale, const float* hyper, cudaStream_t stream) {
  constexpr int kBytes = kThreads / 32 * kStages * static_cast<int>(sizeof(Stage));
  if (!ensure_dynamic_smem(reinterpret_cast<const void*>(adamw8_kernel<COLUMNS>), kBytes)) return -20;
  return launch_code(launch_pdl(adamw8_kernel<COLUMNS>, dim3(t.n_blocks), dim3(kThreads), kBytes, stream, t, s, grad_scale, hyper,
                                addresses_of<COLUMNS>(t)));
}

template <int COLUMNS, class T>
int launch_values(const State8List& t, bool is_signed, T* out, cudaStream_t stream) {
  const auto run = [&](auto* kernel) {
    return launch_code(launch_pdl(kernel, dim3(t.n_blocks), dim3(kThreads), 0, stream, t, out, addresses_of<COLUMNS>(t)));
  };
  return is_signed ? run(state8_values_kernel<T, true, COLUMNS>) : run(state8_values_kernel<T, false, COLUMNS>);
}

}  // namespace

int adamw8_multi(const State8List& t, const Adam8Scalars& s, const float* grad_scale, const float* hyper, cudaStream_t stream) {
  if (t.n_blocks <= 0) return 0;
  if (!fits(t)) return -1;
  return t.host_ptrs ? launch_step<7>(t, s, grad_scale, hyper, stream) : launch_step<0>(t, s, grad_scale, hyper, stream);
}

int state8_values_multi(const State8List& t, bool is_signed, void* out, bool bf16, cudaStream_t stream) {
  if (t.n_blocks <= 0) return 0;
  if (!fits(t)) return -1;
  const auto run = [&](auto* to) { return t.host_ptrs ? launch_values<3>(t, is_signed, to, stream) : launch_values<0>(t, is_signed, to, stream); };
  return bf16 ? run(static_cast<__nv_bfloat16*>(out)) : run(static_cast<float*>(out));
}

}  // namespace tb
