// frn_prompt_attention.cu -- causal grouped-query attention over packed
// prompts.
//
//   out[i, h, :] = sum_{j <= i} softmax_j(scale * q[i, h, :] . k[j, h / G, :]) v[j, h / G, :]
//
// for every token i of every sequence, j running over the tokens of the same
// sequence; the sequences lie one after the other in the token dimension,
// sequence b in rows [cu_seqlens[b], cu_seqlens[b + 1]).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

#include "frn_internal.h"
#include "frn_ptx.cuh"

namespace frn {

// One warp per (token, query head): lanes hold the head dims, one key a step.
template <typename T, int DQK, int DV>
__global__ void __launch_bounds__(128) prompt_attention_kernel(const PromptProblem p) {
  constexpr int EQ = DQK / 32, EV = DV / 32;
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= p.tokens * p.Hq) return;
  const int64_t i = row / p.Hq, h = row % p.Hq, kvh = h / (p.Hq / p.Hkv);
  int64_t first = -1;
  for (int64_t b = 0; b < p.batch; ++b) {
    const int64_t from = p.cu_seqlens[b], to = p.cu_seqlens[b + 1];
    if (from < 0 || to > p.tokens || to - from > p.max_seqlen)
      atomicOr(&g_frn_device_error, kDevErrBadLength);
    if (from >= 0 && from <= i && i < to && i < from + p.max_seqlen) first = from;
  }
  if (first < 0) return;
  const T* q = static_cast<const T*>(p.q) + i * p.q_token_stride + h * p.q_head_stride;
  float qf[EQ], acc[EV];
#pragma unroll
  for (int e = 0; e < EQ; ++e)
    qf[e] = static_cast<float>(q[lane + 32 * e]) * p.scale * 1.4426950408889634f;
#pragma unroll
  for (int e = 0; e < EV; ++e) acc[e] = 0.f;
  float m = -FLT_MAX, l = 0.f;
  for (int64_t j = first; j <= i; ++j) {
    const T* k = static_cast<const T*>(p.k) + j * p.k_token_stride + kvh * p.k_head_stride;
    const T* v = static_cast<const T*>(p.v) + j * p.v_token_stride + kvh * p.v_head_stride;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < EQ; ++e) s = fmaf(qf[e], static_cast<float>(k[lane + 32 * e]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float m_new = fmaxf(m, s), c = exp2f(m - m_new), w = exp2f(s - m_new);
    m = m_new;
    l = l * c + w;
#pragma unroll
    for (int e = 0; e < EV; ++e) acc[e] = fmaf(w, static_cast<float>(v[lane + 32 * e]), acc[e] * c);
  }
  T* out = static_cast<T*>(p.out) + i * p.out_token_stride + h * p.out_head_stride;
#pragma unroll
  for (int e = 0; e < EV; ++e) out[lane + 32 * e] = static_cast<T>(acc[e] / l);
}

template <typename T, int DQK, int DV>
static int launch_prompt(const PromptProblem& g, cudaStream_t stream) {
  prompt_attention_kernel<T, DQK, DV>
      <<<static_cast<unsigned>((g.tokens * g.Hq + 3) / 4), 128, 0, stream>>>(g);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("launch prompt_attention", e);
  return 0;
}

template <typename T>
static int launch_prompt_d(const PromptProblem& g, cudaStream_t s) {
  if (g.Dqk == 192) return launch_prompt<T, 192, 128>(g, s);
  if (g.Dqk == 128) return launch_prompt<T, 128, 128>(g, s);
  return launch_prompt<T, 64, 64>(g, s);
}

int run_prompt_attention(const PromptProblem& g, cudaStream_t s) {
  return g.dtype == FRN_DTYPE_BF16 ? launch_prompt_d<__nv_bfloat16>(g, s)
                                   : launch_prompt_d<__half>(g, s);
}

}  // namespace frn
