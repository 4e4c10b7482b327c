// kv4_attention.cu — attention over the paged 4-bit KV cache (kv4.cuh): query row i of a sequence of length L with n
// rows sees keys 0 .. L - n + i, out = sum_t p_t v_t / sum_t p_t with p_t = 2^(q . k_t - m), one pass over the keys with
// a running maximum; k and v are scale * code + bias per group of 64 dims.
//
// One CTA of 4 warps per (sequence, row, head), a warp a key at a time.
#include <cfloat>

#include "kv4.cuh"

namespace agxc {
namespace {

struct Kv4AttnParams {
  Kv4 c;
  const void* q;
  void* out;
  int bf16, B, n, H, table_ld, max_pages;
  const int32_t* table;
  const int32_t* lengths;
  unsigned* err;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <int HD, typename T>
__global__ void __launch_bounds__(128) kv4_attn_simple(const __grid_constant__ Kv4AttnParams p) {
  using Tile = Kv4Tile<HD>;
  constexpr int E = HD / 32;
  const int h = blockIdx.x % p.H, i = blockIdx.x / p.H % p.n, b = blockIdx.x / p.H / p.n;
  const int j = h / (p.H / p.c.kvh), warp = threadIdx.x >> 5, l = threadIdx.x & 31;
  int len = p.lengths[b];
  const int64_t most = static_cast<int64_t>(p.max_pages) * p.c.page;
  if (len < 0 || len > most) {
    if (threadIdx.x == 0) atomicOr(p.err, kErrBadPos);
    len = len < 0 ? 0 : static_cast<int>(most);
  }
  const int keys = len - p.n + i + 1;
  const int64_t row = (static_cast<int64_t>(b) * p.n + i) * p.H + h;
  float q[E], o[E] = {}, m = -FLT_MAX, sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = to_f(static_cast<const T*>(p.q)[row * HD + l * E + e]);
  const int g = l * E / 64, byte = l * E % 64 / 2;
  for (int t = warp; t < keys; t += 4) {
    const int page = p.table[static_cast<int64_t>(b) * p.table_ld + t / p.c.page], tt = t & 15;
    if (page < 0 || page >= p.c.pages) {
      if (l == 0) atomicOr(p.err, kErrBadPos);
      continue;
    }
    const uint8_t* tile = Tile::ptr(p.c, page, j, t % p.c.page >> 4);
    const __half2* sb = reinterpret_cast<const __half2*>(tile + Tile::kSb + tt * Tile::kEntry);
    const float2 ks = __half22float2(sb[g]), vs = __half22float2(sb[Tile::G + g]);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const unsigned c = tile[Tile::k_at(tt, g, byte + e / 2)] >> (4 * (e & 1)) & 15;
      s += q[e] * (static_cast<float>(c) * ks.x + ks.y);
    }
    s = warp_sum(s);
    const float mn = fmaxf(m, s), f = exp2f(m - mn), w = exp2f(s - mn);
    m = mn;
    sum = sum * f + w;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const unsigned c = tile[Tile::v_at(tt, g, byte + e / 2)] >> (4 * (e & 1)) & 15;
      o[e] = o[e] * f + w * (static_cast<float>(c) * vs.x + vs.y);
    }
  }
  __shared__ float so[4][HD], sm[4], ss[4];
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][l * E + e] = o[e];
  if (l == 0) {
    sm[warp] = m;
    ss[warp] = sum;
  }
  __syncthreads();
  const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float den = 0.f;
  for (int w = 0; w < 4; ++w) den += ss[w] * exp2f(sm[w] - mm);
  for (int d = threadIdx.x; d < HD; d += 128) {
    float v = 0.f;
    for (int w = 0; w < 4; ++w) v += so[w][d] * exp2f(sm[w] - mm);
    static_cast<T*>(p.out)[row * HD + d] = static_cast<T>(den > 0.f ? v / den : 0.f);
  }
}

int attn_check(const agxc_kv4_attention_args* a) {
  if (!a) return fail(AGXC_EINVAL, "kv4_attention: null argument");
  if (int rc = kv4_check(&a->cache, "kv4_attention")) return rc;
  if (a->dtype != AGXC_F16 && a->dtype != AGXC_BF16) return fail(AGXC_EINVAL, "kv4_attention: q fp16 or bf16");
  if (a->batch < 0 || a->rows < 0) return fail(AGXC_EINVAL, "kv4_attention: batch and rows >= 0");
  if (a->heads < 1 || a->heads % a->cache.kv_heads)
    return fail(AGXC_EINVAL, "kv4_attention: heads a positive multiple of kv_heads");
  if (a->max_pages < 0 || a->table_ld < a->max_pages)
    return fail(AGXC_EINVAL, "kv4_attention: 0 <= max_pages <= table_ld");
  if (static_cast<int64_t>(a->max_pages) * a->cache.page_size > 0x7fffff00)
    return fail(AGXC_EINVAL, "kv4_attention: max_pages * page_size must stay below 2^31");
  if (static_cast<int64_t>(a->batch) * a->rows * a->heads > 0x7fffffff)
    return fail(AGXC_EINVAL, "kv4_attention: too many query rows for one call");
  return 0;
}

}  // namespace
}  // namespace agxc

using namespace agxc;

extern "C" {

AGXC_API int64_t agxc_kv4_attention_workspace(agxc_ctx* ctx, const agxc_kv4_attention_args* a) {
  if (!ctx) return fail(AGXC_EINVAL, "kv4_attention: null context");
  if (attn_check(a)) return -1;
  return 0;
}

AGXC_API int agxc_kv4_attention_dev(agxc_ctx* ctx, const agxc_kv4_attention_args* a, void* stream) {
  if (!ctx) return fail(AGXC_EINVAL, "kv4_attention: null context");
  if (int rc = attn_check(a)) return rc;
  if (a->batch == 0 || a->rows == 0) return 0;
  if (!a->q_dev || !a->out_dev || !a->lengths_dev || (a->max_pages && !a->page_table_dev))
    return fail(AGXC_EINVAL, "kv4_attention: null buffer");
  if (reinterpret_cast<uintptr_t>(a->q_dev) % 16 || reinterpret_cast<uintptr_t>(a->out_dev) % 16)
    return fail(AGXC_EINVAL, "kv4_attention: q and out must be 16-byte aligned");
  Kv4AttnParams p;
  p.c = kv4_of(a->cache);
  p.q = a->q_dev; p.out = a->out_dev; p.bf16 = a->dtype == AGXC_BF16; p.B = a->batch; p.n = a->rows; p.H = a->heads;
  p.table_ld = a->table_ld; p.max_pages = a->max_pages; p.table = a->page_table_dev; p.lengths = a->lengths_dev;
  p.err = ctx->err_dev;
  cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const unsigned grid = static_cast<unsigned>(a->batch) * a->rows * a->heads;
  if (a->cache.head_dim == 128) {
    if (p.bf16) kv4_attn_simple<128, __nv_bfloat16><<<grid, 128, 0, s>>>(p);
    else kv4_attn_simple<128, __half><<<grid, 128, 0, s>>>(p);
  } else {
    if (p.bf16) kv4_attn_simple<64, __nv_bfloat16><<<grid, 128, 0, s>>>(p);
    else kv4_attn_simple<64, __half><<<grid, 128, 0, s>>>(p);
  }
  AGXC_CUDA(cudaGetLastError());
  return 0;
}

}  // extern "C"
