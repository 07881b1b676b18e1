// Host-callable launchers of the mixture-of-experts kernels and of the 8-bit activation checkpoints (raw pointers, sizes, a stream).
// Each returns 0, or a negative code for sizes or addresses it does not take and for a launch that was refused.
//
// Rows grouped by expert: row r belongs to the expert e with offsets[e] <= r < offsets[e + 1]; offsets has E + 1 entries, starts at 0
// and does not decrease; rows from offsets[E] on belong to none.  The kernels clamp what they read from `offsets` to [0, R], and skip
// slots and rows outside their matrices: wrong values give wrong results, never an access outside a tensor.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tb {

constexpr int kMaxExperts = 384;
constexpr int kMaxChoices = 16;
constexpr int kActBlock = 64;      // values of a row that share a scale in an 8-bit checkpoint

// ---- router (moe_route.cu) ------------------------------------------------------------------------
// Choices of one row of logits: the k largest, ties to the lowest index; a choice whose logit is -inf is not made.
// weights [T, k], experts [T, k], slots [T, k] (row of the choice, -1: not made or beyond the capacity), offsets [E + 1],
// rows [T k] (t k + j of each row, -1 behind offsets[E]), counts [E] (choices made, before the capacity), aux [1].
// scratch: route_scratch_ints(T, E, how) 32-bit words.  capacity 0: no limit.
// how (nullptr: the logits choose, weights are the softmax over the chosen): choice by scores, see moe_route.cu.
constexpr int kMaxExpertGroups = 32;
struct RouteScore {
  bool sigmoid;            // else softmax
  const float* bias;       // [E], nullptr: none
  int groups, top_groups;  // experts in `groups` equal parts, `top_groups` of which stay open to a token
  bool normalize;          // weights over their sum
  float scale;             // times this, not 0
  int group_scores;        // a group counts by its so many largest, 1 or 2
};
int64_t route_scratch_ints(int T, int E, const RouteScore* how);
int route_kernels(int T, int E, const RouteScore* how);      // that route_fwd launches
[[nodiscard]] int route_fwd(const void* logits, bool bf16, int64_t ld, int T, int E, int k, int capacity, const RouteScore* how,
                            float* weights, int* experts, int* slots, int* offsets, int* rows, int* counts, float* aux, int* scratch,
                            cudaStream_t stream);
// dlogits [T, E] (the logits' type) from dweights [T, k] (nullptr: none) and daux [1] (nullptr: none)
[[nodiscard]] int route_bwd(const void* logits, bool bf16, int64_t ld, const float* weights, const int* experts, const int* counts,
                            const float* dweights, const float* daux, void* dlogits, int T, int E, int k, const RouteScore* how,
                            cudaStream_t stream);      // (of `how` the bias and the groups are not looked at)
// bias[e] += rate sign(mean of counts - counts[e])
[[nodiscard]] int balance_bias(float* bias, const int* counts, int E, float rate, cudaStream_t stream);

// ---- rows to expert order and back (moe_rows.cu) -----------------------------------------------------
// out[r] = bf16(x[rows[r] / k]), zeros where rows[r] < 0
[[nodiscard]] int rows_gather(const void* x, bool x_bf16, int64_t ldx, const int* rows, __nv_bfloat16* out, int T, int k, int R, int D,
                              cudaStream_t stream);
// out[t] = sum_j weights[t, j] y[slots[t, j]] (weights nullptr: 1), fp32 sums in the order of the choices
[[nodiscard]] int rows_combine(const void* y, bool y_bf16, const float* weights, const int* slots, void* out, bool out_bf16, int T, int k,
                               int R, int D, cudaStream_t stream);
// dy[slots[t, j]] = bf16(weights[t, j] dout[t]), zeros in rows of no choice; dweights[t, j] = <y[slot], dout[t]>, 0 without a slot
[[nodiscard]] int rows_combine_bwd(const void* dout, bool dout_bf16, int64_t ld, const __nv_bfloat16* y, const float* weights,
                                   const int* slots, const int* offsets, __nv_bfloat16* dy, float* dweights, int T, int k, int E, int D,
                                   cudaStream_t stream);

// ---- products grouped by expert (grouped_gemm_sm100.cu) ------------------------------------------------
// y[r] = x[r] W[e(r)]^T (w_t false, W [E, N, K]) or x[r] W[e(r)] (w_t true, W [E, K, N]); rows of no expert: zeros.  x [R, K].
[[nodiscard]] int grouped_gemm(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* w, bool w_t, const int* offsets, __nv_bfloat16* y,
                               int R, int E, int N, int K, int* err, int num_sms, cudaStream_t stream);
// The same with w_t false and y in fp32, for few rows per expert only (grouped_gemm_few): y is added up over a token's choices afterwards,
// and costs next to nothing there.  early (here and below): the kernel before on the stream is one of the same feed-forward pass, so that all
// that was there before the pass has ended and nothing that still runs writes w; the kernel may then read w before that one has ended.
bool grouped_gemm_few(int R, int E);
[[nodiscard]] int grouped_gemm_f32(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* w, const int* offsets, float* y, int R, int E,
                                   int N, int K, bool early, int* err, int num_sms, cudaStream_t stream);
// act [R, F] = silu(g) u of g | u = x W[e]^T, W [E, 2F, K] = gate rows over up rows.  Gate and up go to gu [R, 2F] in bf16, or to q
// [R, 2F] and scales [R, 2 ceil(F / 64)] in 8 bits, or nowhere; rows of no expert: zeros.
// list (nullptr: the R rows of x are in expert order): row r is row list[r] / k of the `count` rows of x, what `rows` of route_fwd says.
// Only where grouped_swiglu_listed, and not with q.
bool grouped_swiglu_listed(int R, int E);
[[nodiscard]] int grouped_swiglu(const __nv_bfloat16* x, int64_t ldx, const int* list, int k, int count, const __nv_bfloat16* w,
                                 const int* offsets, __nv_bfloat16* act, __nv_bfloat16* gu, int8_t* q, float* scales, int R, int E, int F,
                                 int K, bool early, int* err, int num_sms, cudaStream_t stream);
// dw[e] [N, K] = sum over the rows of e of dy[r]^T x[r], bf16 or fp32; zeros for an expert without rows
[[nodiscard]] int grouped_wgrad(const __nv_bfloat16* dy, int64_t lddy, const __nv_bfloat16* x, int64_t ldx, const int* offsets, void* dw,
                                bool dw_bf16, int R, int E, int N, int K, int* err, int num_sms, cudaStream_t stream);

// ---- the whole feed-forward of a few tokens, without gradients (moe_token.cu) ---------------------------
constexpr int kTokenTokens = 4, kTokenChoices = 32;      // at most
int64_t token_scratch_bytes(int T, int k, int F);
// out [T, D] (x's type) and aux [1] from logits [T, E] and x [T, D]; scratch: token_scratch_bytes, on 16 bytes
[[nodiscard]] int token_mlp(const void* logits, bool logits_bf16, int64_t ldl, const void* x, bool x_bf16, int64_t ldx,
                            const __nv_bfloat16* w_gate_up, const __nv_bfloat16* w_down, void* out, float* aux, void* scratch, int T, int E,
                            int k, int capacity, int D, int F, cudaStream_t stream);

// ---- 8-bit activation checkpoints (act8.cu) --------------------------------------------------------------
// Per row and block of 64 values: a = the largest magnitude, q = sign(x) floor(127 |x| / a + 1/2), scale = a / 127 (0 for a block of
// zeros, NaN for one that holds a value that is not finite).  q [M, N], scales [M, ceil(N / 64)].
[[nodiscard]] int quantize8(const __nv_bfloat16* x, int64_t ldx, int8_t* q, float* scales, int64_t M, int N, cudaStream_t stream);
[[nodiscard]] int dequantize8(const int8_t* q, const float* scales, __nv_bfloat16* x, int64_t M, int N, cudaStream_t stream);
// act [M, F] = silu(g) u of gu [M, 2F] = g | u; q [M, 2F] and scales [M, 2 ceil(F / 64)]: both halves as quantize8 keeps them (nullptr: not
// kept)
[[nodiscard]] int swiglu8_fwd(const __nv_bfloat16* gu, int64_t ldgu, __nv_bfloat16* act, int8_t* q, float* scales, int64_t M, int F,
                              cudaStream_t stream);
[[nodiscard]] int swiglu8_bwd(const __nv_bfloat16* dact, int64_t ldd, const int8_t* q, const float* scales, __nv_bfloat16* dgu, int64_t M,
                              int F, cudaStream_t stream);
// The experts' SwiGLU backward, over choices i = t k + j with row r = slots[i] and weight w = weights[i]; s [R, F] = dout W_down.
// Gate and up come from gu (bf16) or, where gu is nullptr, from (q, scales).  dgu[r] = d(gate) | d(up) for d(act) = w s,
// act_w[r] = w act, dweights[i] = <act, s>; zeros in rows of no choice, and 0 for a choice without a row.  F a multiple of 8, matrices on
// 16 bytes.
[[nodiscard]] int expert_swiglu_bwd(const __nv_bfloat16* s, const __nv_bfloat16* gu, const int8_t* q, const float* scales,
                                    const float* weights, const int* slots, const int* offsets, __nv_bfloat16* dgu, __nv_bfloat16* act_w,
                                    float* dweights, int R, int E, int F, cudaStream_t stream);

}  // namespace tb
