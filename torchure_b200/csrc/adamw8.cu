// AdamW over many tensors whose two moments are held in 8 bits, one launch, and the moments read back.
//
// A block of 128 consecutive values of a tensor has one fp32 scale.  With a the block's largest magnitude, a magnitude x is brought to
// y = x TOP / a + FIRST and held as y's fp32 pattern cut to 3 bits of mantissa, counted from FIRST's pattern:
//   code = ((bits(y) + (r << 4)) >> 20) - (bits(FIRST) >> 20),   x kept = (value(code) - FIRST) a / TOP
// (even steps next to zero, steps of an eighth further up).  First moment: a sign bit and FIRST = 2^-15, 127 steps down to a 2^-19; second
// moment: FIRST = 2^-31, 255 steps down to a 2^-35, so that its root covers what the first moment covers.  r are 16 random bits: a value goes to
// one of its two neighbours with the probability that makes the mean its own.  To the nearest, a second moment that changes by 1 - beta2 of
// itself a step, less than half a step of the code, would stay where it is for good.  A second moment above zero keeps at least the first step:
// no update divides by eps alone where the gradients have been small beside the block's.
// A block that holds something that is not finite reads back as NaN, one whose largest magnitude is under 2^-100 as zeros.
//
// Random bits: h(i) = mix(key ^ low 32 bits of i), key from (seed, step, tensor, high bits of i), mix two rounds of xorshift and multiplication
// (constants by C. Wellons, 2018); 16 bits for each moment.
//
// Arithmetic is fp32, every operation rounded by itself in the order written (no contraction): the result is that of the same statements in plain
// tensor operations, bit for bit, and two replicas stay equal.
//
// Bound by memory: an element reads 4 + 4 + 1 + 1 bytes and writes 4 + 1 + 1 (+ 2 of the bf16 shadow), 18.1 with the scales, against 30 with the
// moments in fp32.
#include "api.h"
#include "common.cuh"

namespace tb {

namespace {

constexpr int kThreads = 512;
constexpr float kFirstM = 3.0517578125e-05f, kFirstV = 4.656612873077393e-10f;      // 2^-15, 2^-31
constexpr int kKeyM = 896, kKeyV = 768;                                             // their patterns >> 20
constexpr float kTopM = 1.875f - 3.0517578125e-05f, kTopV = 1.875f;
constexpr float kTinyBlock = 7.888609052210118e-31f;      // 2^-100

__host__ __device__ constexpr uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x7feb352du;
  x = (x ^ (x >> 15)) * 0x846ca68bu;
  return x ^ (x >> 16);
}

template <bool SIGNED>
__device__ __forceinline__ float decode8(uint32_t code, float scale) {
  const uint32_t size = SIGNED ? code & 127u : code;
  const float y = __uint_as_float((size + (SIGNED ? kKeyM : kKeyV)) << 20) - (SIGNED ? kFirstM : kFirstV);
  const float x = __fmul_rn(y, scale);
  return SIGNED && (code & 128u) ? -x : x;
}

struct Coder {
  float scale, inverse;
  bool fine;
};
template <bool SIGNED>
__device__ __forceinline__ Coder coder_for(float top) {
  constexpr float kTop = SIGNED ? kTopM : kTopV;
  Coder c;
  c.fine = top >= kTinyBlock && top < INFINITY;
  c.inverse = __fmul_rn(__frcp_rn(top), kTop);
  c.scale = c.fine ? __fmul_rn(top, static_cast<float>(1.0 / static_cast<double>(kTop))) : top < kTinyBlock ? 0.f : __uint_as_float(0x7fc00000u);
  return c;
}
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode8(float x, const Coder& c, uint32_t r) {
  const float y = __fadd_rn(__fmul_rn(fabsf(x), c.inverse), SIGNED ? kFirstM : kFirstV);
  int code = static_cast<int>((__float_as_uint(y) + (r << 4)) >> 20) - (SIGNED ? kKeyM : kKeyV);
  code = min(code, SIGNED ? 127 : 255);
  if (SIGNED) code += x < 0.f ? 128 : 0;
  else if (x > 0.f) code = max(code, 1);
  return c.fine ? static_cast<uint32_t>(code) : 0u;
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

// A warp per block of 128, four values a thread
__global__ void __launch_bounds__(kThreads)
adamw8_kernel(State8List t, Adam8Scalars s, const float* __restrict__ grad_scale, const float* __restrict__ hyper) {
  pdl_wait();
  pdl_launch_dependents();
  uint32_t key = s.key;
  if (hyper) {      // what changes from step to step read from device memory: the launch can be replayed from a graph
    s.step_size = hyper[0];
    s.root = hyper[1];
    s.decay = hyper[2];
    key = __float_as_uint(hyper[3]);
  }
  const int ti = t.block_tensor[blockIdx.x], n_tensors = t.n_tensors;
  const int64_t n = t.numel[ti], lo = static_cast<int64_t>(t.block_chunk[blockIdx.x]) * kChunkElems;
  const int64_t hi = lo + kChunkElems < n ? lo + kChunkElems : n;
  const int64_t* ptr = t.ptrs + ti;
  float* p = reinterpret_cast<float*>(ptr[0]);
  const void* g = reinterpret_cast<const void*>(ptr[n_tensors]);
  uint8_t* m = reinterpret_cast<uint8_t*>(ptr[2 * n_tensors]);
  uint8_t* v = reinterpret_cast<uint8_t*>(ptr[3 * n_tensors]);
  float* m_scale = reinterpret_cast<float*>(ptr[4 * n_tensors]);
  float* v_scale = reinterpret_cast<float*>(ptr[5 * n_tensors]);
  __nv_bfloat16* sh = reinterpret_cast<__nv_bfloat16*>(ptr[6 * n_tensors]);
  const bool g16 = (t.flags[ti] & 1) != 0;
  const bool vp = on(p, 16), vg = on(g, g16 ? 8 : 16), vm = on(m, 4), vv = on(v, 4), vs = on(sh, 8);
  float gs = grad_scale ? *grad_scale : 1.f;
  if (s.maximize) gs = -gs;
  key = mix32(key + 0x85ebca6bu * static_cast<uint32_t>(ti) + 0xc2b2ae35u * static_cast<uint32_t>(lo >> 32));
  const int lane = threadIdx.x & 31;
#pragma unroll 2
  for (int64_t b = lo + (threadIdx.x >> 5) * kStateBlock; b < hi; b += (kThreads / 32) * kStateBlock) {
    const int64_t i = b + lane * 4;
    const int left = static_cast<int>(hi - i < 4 ? (hi - i > 0 ? hi - i : 0) : 4);
    float px[4], gx[4], mx[4], vx[4];
    load4(p + i, vp, left, px);
    if (g16) load4(static_cast<const __nv_bfloat16*>(g) + i, vg, left, gx);
    else load4(static_cast<const float*>(g) + i, vg, left, gx);
    const uint32_t mc = load_codes(m + i, vm, left), vc = load_codes(v + i, vv, left);
    const float ms = m_scale[b / kStateBlock], vscale = v_scale[b / kStateBlock];
    uint32_t m_top = 0, v_top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gj = __fmul_rn(gx[j], gs);
      mx[j] = __fadd_rn(__fmul_rn(decode8<true>((mc >> (8 * j)) & 255u, ms), s.beta1), __fmul_rn(gj, s.rest1));
      vx[j] = __fadd_rn(__fmul_rn(decode8<false>((vc >> (8 * j)) & 255u, vscale), s.beta2), __fmul_rn(__fmul_rn(gj, s.rest2), gj));
      const float denom = __fadd_rn(__fmul_rn(__fsqrt_rn(vx[j]), s.root), s.eps);
      px[j] = __fsub_rn(__fmul_rn(px[j], s.decay), __fmul_rn(__fdiv_rn(mx[j], denom), s.step_size));
      if (j < left) {
        m_top = max(m_top, __float_as_uint(fabsf(mx[j])));      // (patterns of magnitudes are ordered as they are; NaN last)
        v_top = max(v_top, __float_as_uint(fabsf(vx[j])));
      }
    }
    store4(p + i, vp, left, px);
    if (sh) store4(sh + i, vs, left, px);
    const Coder cm = coder_for<true>(__uint_as_float(__reduce_max_sync(0xffffffffu, m_top)));
    const Coder cv = coder_for<false>(__uint_as_float(__reduce_max_sync(0xffffffffu, v_top)));
    uint32_t mo = 0, vo = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t h = mix32(key ^ static_cast<uint32_t>(i + j));
      mo |= encode8<true>(mx[j], cm, h & 0xffffu) << (8 * j);
      vo |= encode8<false>(vx[j], cv, h >> 16) << (8 * j);
    }
    store_codes(m + i, vm, left, mo);
    store_codes(v + i, vv, left, vo);
    if (lane == 0) {
      m_scale[b / kStateBlock] = cm.scale;
      v_scale[b / kStateBlock] = cv.scale;
    }
  }
}

// ptrs: codes, scales, and the values' place in `all`, in elements
template <class T, bool SIGNED>
__global__ void __launch_bounds__(kThreads)
state8_values_kernel(State8List t, T* __restrict__ all) {
  pdl_wait();
  pdl_launch_dependents();
  const int ti = t.block_tensor[blockIdx.x];
  const int64_t n = t.numel[ti], lo = static_cast<int64_t>(t.block_chunk[blockIdx.x]) * kChunkElems;
  const int64_t hi = lo + kChunkElems < n ? lo + kChunkElems : n;
  const uint8_t* codes = reinterpret_cast<const uint8_t*>(t.ptrs[ti]);
  const float* scales = reinterpret_cast<const float*>(t.ptrs[t.n_tensors + ti]);
  T* out = all + t.ptrs[2 * t.n_tensors + ti];
  const bool vc = on(codes, 4), vo = on(out, 4 * sizeof(T));
#pragma unroll 4
  for (int64_t i = lo + threadIdx.x * 4; i < hi; i += kThreads * 4) {
    const int left = static_cast<int>(hi - i < 4 ? hi - i : 4);
    const uint32_t c = load_codes(codes + i, vc, left);
    const float scale = scales[i / kStateBlock];
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t code = (c >> (8 * j)) & 255u;
      x[j] = decode8<SIGNED>(code, scale);
    }
    store4(out + i, vo, left, x);
  }
}

}  // namespace

int adamw8_multi(const State8List& t, const Adam8Scalars& s, const float* grad_scale, const float* hyper, cudaStream_t stream) {
  if (t.n_blocks <= 0) return 0;
  return launch_code(launch_pdl(adamw8_kernel, dim3(t.n_blocks), dim3(kThreads), 0, stream, t, s, grad_scale, hyper));
}

int state8_values_multi(const State8List& t, bool is_signed, void* out, bool bf16, cudaStream_t stream) {
  if (t.n_blocks <= 0) return 0;
  const dim3 grid(t.n_blocks), block(kThreads);
  const auto run = [&](auto* kernel, auto* to) { return launch_code(launch_pdl(kernel, grid, block, 0, stream, t, to)); };
  if (bf16)
    return is_signed ? run(state8_values_kernel<__nv_bfloat16, true>, static_cast<__nv_bfloat16*>(out))
                     : run(state8_values_kernel<__nv_bfloat16, false>, static_cast<__nv_bfloat16*>(out));
  return is_signed ? run(state8_values_kernel<float, true>, static_cast<float*>(out))
                   : run(state8_values_kernel<float, false>, static_cast<float*>(out));
}

}  // namespace tb
