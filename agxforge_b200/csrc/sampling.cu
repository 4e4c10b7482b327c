// sampling.cu — one token a row from logits, with temperature, top-k, top-p and min-p, at given uniform numbers.
//
// Weights are w = floor(2^40 exp((l - max) / T)) as 64-bit integers, so a row's sums are exact whatever their order and
// the token does not depend on how the row is split. Tokens are ranked by a 64-bit key, the logit's order in the high
// half and the index (lower first) in the low half; top-k and top-p each keep the keys from some key up, min-p compares
// exp((l - max) / T) itself, and the token is the first kept index whose cumulative weight exceeds floor(u * total).
//
// One CTA a row; each cut is found bit by bit, one pass over the row a bit.
#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace agxc {
namespace {

struct SampleParams {
  const void* x;
  int64_t ld;
  int B, V;
  const float* u;
  float T, top_p, min_p;
  int top_k;
  const float* T_a;
  const int32_t* k_a;
  const float* p_a;
  const float* m_a;
  int32_t* token;
  float* prob;
};

constexpr int kThreads = 1024;
constexpr float kOne = 1099511627776.f;  // 2^40

template <int DT>
__device__ __forceinline__ float logit(const void* x, int64_t i) {
  float v;
  if (DT == AGXC_F32) v = static_cast<const float*>(x)[i];
  else if (DT == AGXC_F16) v = __half2float(static_cast<const __half*>(x)[i]);
  else v = __bfloat162float(static_cast<const __nv_bfloat16*>(x)[i]);
  return v != v ? -INFINITY : v + 0.f;  // + 0: the two zeros rank alike
}

// larger logits first, then lower indices: the larger key ranks first
__device__ __forceinline__ uint64_t rank_key(float v, int i) {
  const uint32_t b = __float_as_uint(v);
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<uint64_t>(o) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

struct Row {
  float best, inv_t;
  bool greedy;
  __device__ float e(float v) const {
    if (v == -INFINITY) return 0.f;
    const float d = v == best ? 0.f : __fsub_rn(v, best);
    return greedy ? (d == 0.f ? 1.f : 0.f) : expf(__fmul_rn(d, inv_t));
  }
};

__device__ __forceinline__ int64_t weight(float e) { return __float2ll_rz(e * kOne); }

__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* sh) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t t = 0;
  for (int w = 0; w < kThreads / 32; ++w) t += sh[w];
  return t;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleParams p) {
  const int b = blockIdx.x, V = p.V;
  const int64_t base = static_cast<int64_t>(b) * p.ld;
  __shared__ int64_t sh[32];
  __shared__ float shf[32];
  __shared__ int found;
  const float T = p.T_a ? p.T_a[b] : p.T, top_p = p.p_a ? p.p_a[b] : p.top_p, min_p = p.m_a ? p.m_a[b] : p.min_p;
  const int top_k = p.k_a ? p.k_a[b] : p.top_k;
  float best = -INFINITY;
  for (int i = threadIdx.x; i < V; i += kThreads) best = fmaxf(best, logit<DT>(p.x, base + i));
  best = warp_max(best);
  if ((threadIdx.x & 31) == 0) shf[threadIdx.x >> 5] = best;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) best = fmaxf(best, shf[w]);
  if (best == -INFINITY) {
    if (threadIdx.x == 0) {
      p.token[b] = -1;
      if (p.prob) p.prob[b] = 0.f;
    }
    return;
  }
  Row r;
  r.best = best;
  r.greedy = T == 0.f;
  r.inv_t = r.greedy ? 1.f : __fdiv_rn(1.f, T);
  uint64_t cut = 0;  // keys from `cut` up are kept
  if (top_k > 0 && top_k < V) {
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t at = cut | 1ull << bit;
      int64_t n = 0;
      for (int i = threadIdx.x; i < V; i += kThreads) n += rank_key(logit<DT>(p.x, base + i), i) >= at;
      if (block_sum(n, sh) >= top_k) cut = at;
    }
  }
  if (top_p < 1.f) {
    const uint64_t from = cut;
    int64_t n = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float v = logit<DT>(p.x, base + i);
      if (rank_key(v, i) >= from) n += weight(r.e(v));
    }
    const int64_t total = block_sum(n, sh);
    const double bar = ceil(__dmul_rn(static_cast<double>(top_p), static_cast<double>(total)));
    const int64_t need = bar > 1.0 ? static_cast<int64_t>(bar) : 1;
    cut = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t at = cut | 1ull << bit, lo = at > from ? at : from;
      n = 0;
      for (int i = threadIdx.x; i < V; i += kThreads) {
        const float v = logit<DT>(p.x, base + i);
        if (rank_key(v, i) >= lo) n += weight(r.e(v));
      }
      if (block_sum(n, sh) >= need) cut = at;
    }
  }
  auto kept = [&](int i) -> int64_t {
    const float v = logit<DT>(p.x, base + i);
    const float e = r.e(v);
    return rank_key(v, i) >= cut && e >= min_p ? weight(e) : 0;
  };
  int64_t n = 0;
  for (int i = threadIdx.x; i < V; i += kThreads) n += kept(i);
  const int64_t total = block_sum(n, sh);
  if (total == 0) {
    if (threadIdx.x == 0) {
      p.token[b] = -1;
      if (p.prob) p.prob[b] = 0.f;
    }
    return;
  }
  const double u = r.greedy ? 0.0 : static_cast<double>(p.u[b]);
  int64_t target = static_cast<int64_t>(floor(__dmul_rn(u, static_cast<double>(total))));
  target = target < total - 1 ? target : total - 1;
  // each thread a contiguous range of indices; the threads before it in order
  const int per = (V + kThreads - 1) / kThreads, i0 = min(V, static_cast<int>(threadIdx.x) * per), i1 = min(V, i0 + per);
  n = 0;
  for (int i = i0; i < i1; ++i) n += kept(i);
  int64_t up = n;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, up, m);
    if ((threadIdx.x & 31) >= m) up += o;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 31) sh[threadIdx.x >> 5] = up;
  __syncthreads();
  for (int w = 0; w < static_cast<int>(threadIdx.x >> 5); ++w) up += sh[w];
  if (target < up && target >= up - n) {
    int64_t c = up - n;
    for (int i = i0; i < i1; ++i) {
      const int64_t w = kept(i);
      c += w;
      if (c > target) {
        p.token[b] = i;
        if (p.prob)
          p.prob[b] = r.greedy ? 1.f : static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
        break;
      }
    }
  }
}

}  // namespace
}  // namespace agxc

using namespace agxc;

extern "C" AGXC_API int agxc_sample_dev(agxc_ctx* ctx, const agxc_sample_args* a, void* stream) {
  if (!ctx || !a) return fail(AGXC_EINVAL, "sample: null argument");
  if (a->dtype < AGXC_F32 || a->dtype > AGXC_BF16) return fail(AGXC_EINVAL, "sample: logits fp32, fp16 or bf16");
  if (a->batch < 0 || a->vocab < 1) return fail(AGXC_EINVAL, "sample: batch >= 0 and a vocabulary of at least one");
  if (a->logits_ld < a->vocab) return fail(AGXC_EINVAL, "sample: logits_ld < vocab");
  if (!a->temperature_dev && !(a->temperature >= 0.f)) return fail(AGXC_EINVAL, "sample: temperature >= 0");
  if (a->batch == 0) return 0;
  if (!a->logits_dev || !a->u_dev || !a->token_dev) return fail(AGXC_EINVAL, "sample: null buffer");
  SampleParams p;
  p.x = a->logits_dev; p.ld = a->logits_ld; p.B = a->batch; p.V = a->vocab; p.u = a->u_dev;
  p.T = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
  p.T_a = a->temperature_dev; p.k_a = a->top_k_dev; p.p_a = a->top_p_dev; p.m_a = a->min_p_dev;
  p.token = a->token_dev; p.prob = a->prob_dev;
  cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  if (a->dtype == AGXC_F32) sample_kernel<AGXC_F32><<<a->batch, kThreads, 0, s>>>(p);
  else if (a->dtype == AGXC_F16) sample_kernel<AGXC_F16><<<a->batch, kThreads, 0, s>>>(p);
  else sample_kernel<AGXC_BF16><<<a->batch, kThreads, 0, s>>>(p);
  AGXC_CUDA(cudaGetLastError());
  return 0;
}
