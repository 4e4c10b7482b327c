// kv4.cu — the paged 4-bit KV cache's append and read-back (the attention over it is kv4_attention.cu).
//
//   append   x = qkv + bias; optional RMS norm of each q and k head; RoPE on (i, i + hd/2): o1 = x1 c - x2 s,
//            o2 = x2 c + x1 s, each product and sum rounded (as the fp16 cache's append); q = o * qscale, rounded;
//            k and v quantised per 64 dims: scale = (max - min) fp32(1 / 15) and bias = min in fp16 (scale 1 where all are
//            equal), code = rint((x - b) / s) clipped to 0..15, 0 where that is not finite; each step an IEEE fp32
//            operation, so the codes do not depend on how the tokens are batched.
//   rows     scale * code + bias of given slots, one fused multiply-add, rounded to fp16.
#include "kv4.cuh"

namespace agxc {
namespace {

struct AppendParams {
  Kv4 c;
  const void* qkv;
  int64_t ld;
  int dtype, T, H, table_rows;
  const int32_t* pos;
  const int64_t* slots;
  const float* cos_t;
  const float* sin_t;
  const __half* bias;
  const __half* qn;
  const __half* kn;
  float eps, qscale;
  void* q;
  int q_bf16;
  unsigned* err;
};

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if (DT == AGXC_F32) return static_cast<const float*>(p)[i];
  if (DT == AGXC_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// min and max over the LPH lanes of a head
template <int LPH>
__device__ __forceinline__ void head_minmax(float& lo, float& hi) {
#pragma unroll
  for (int m = LPH / 2; m >= 1; m >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
  }
}

__device__ __forceinline__ unsigned code4(float x, float s, float b) {
  const float q = rintf(__fdiv_rn(__fsub_rn(x, b), s));
  return isfinite(q) ? static_cast<unsigned>(fminf(fmaxf(q, 0.f), 15.f)) : 0u;
}

// hd / 4 lanes a head: lane l holds dims 2l, 2l + 1 and the dims hd / 2 above them (a RoPE pair each, and one code byte
// each). A warp takes one head of 128 or two of 64.
template <int HD, int DT>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
  using Tile = Kv4Tile<HD>;
  constexpr int LPH = HD / 4;
  const int heads = p.H + 2 * p.c.kvh;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LPH;
  const int l = threadIdx.x % LPH;
  const bool live = item < static_cast<int64_t>(p.T) * heads;
  const int t = live ? static_cast<int>(item / heads) : 0, head = live ? static_cast<int>(item % heads) : 0;
  const int pos = p.pos[t];
  const int64_t slot = p.slots[t];
  const bool is_q = head < p.H, is_v = head >= p.H + p.c.kvh;
  const bool bad = pos < 0 || pos >= p.table_rows || slot >= static_cast<int64_t>(p.c.pages) * p.c.page;
  if (live && bad && l == 0 && p.err) atomicOr(p.err, kErrBadPos);
  float x[4];
  const int d0 = 2 * l, d1 = HD / 2 + 2 * l;
  const int64_t row = static_cast<int64_t>(t) * p.ld + static_cast<int64_t>(head) * HD;
  x[0] = load1<DT>(p.qkv, row + d0);
  x[1] = load1<DT>(p.qkv, row + d0 + 1);
  x[2] = load1<DT>(p.qkv, row + d1);
  x[3] = load1<DT>(p.qkv, row + d1 + 1);
  if (p.bias) {
    const __half* b = p.bias + static_cast<int64_t>(head) * HD;
    x[0] = __fadd_rn(x[0], __half2float(b[d0]));
    x[1] = __fadd_rn(x[1], __half2float(b[d0 + 1]));
    x[2] = __fadd_rn(x[2], __half2float(b[d1]));
    x[3] = __fadd_rn(x[3], __half2float(b[d1 + 1]));
  }
  if (p.qn) {
    float sum = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
    for (int m = LPH / 2; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (!is_v) {
      const float r = rsqrtf(sum / static_cast<float>(HD) + p.eps);
      const __half* g = is_q ? p.qn : p.kn;
      x[0] = (x[0] * r) * __half2float(g[d0]);
      x[1] = (x[1] * r) * __half2float(g[d0 + 1]);
      x[2] = (x[2] * r) * __half2float(g[d1]);
      x[3] = (x[3] * r) * __half2float(g[d1 + 1]);
    }
  }
  if (!is_v && !bad) {
    const float* c = p.cos_t + static_cast<int64_t>(pos) * (HD / 2);
    const float* s = p.sin_t + static_cast<int64_t>(pos) * (HD / 2);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x1 = x[e], x2 = x[2 + e], cc = c[d0 + e], ss = s[d0 + e];
      x[e] = __fadd_rn(__fmul_rn(x1, cc), -__fmul_rn(x2, ss));
      x[2 + e] = __fadd_rn(__fmul_rn(x2, cc), __fmul_rn(x1, ss));
    }
  }
  // the shuffles below are the whole warp's
  float lo0 = fminf(x[0], x[1]), hi0 = fmaxf(x[0], x[1]), lo1 = fminf(x[2], x[3]), hi1 = fmaxf(x[2], x[3]);
  if (HD == 64) {
    lo0 = fminf(lo0, lo1);
    hi0 = fmaxf(hi0, hi1);
  }
  head_minmax<LPH>(lo0, hi0);
  if (HD == 128) head_minmax<LPH>(lo1, hi1);
  if (!live || bad) return;
  if (is_q) {
    const int64_t o = (static_cast<int64_t>(t) * p.H + head) * HD;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t at = o + (e < 2 ? d0 + e : d1 + e - 2);
      const float v = __fmul_rn(x[e], p.qscale);
      if (p.q_bf16) static_cast<__nv_bfloat16*>(p.q)[at] = __float2bfloat16_rn(v);
      else static_cast<__half*>(p.q)[at] = __float2half_rn(v);
    }
    return;
  }
  if (slot < 0) return;
  const int j = is_v ? head - p.H - p.c.kvh : head - p.H;
  const int page = static_cast<int>(slot / p.c.page), off = static_cast<int>(slot % p.c.page), tt = off & 15;
  uint8_t* tile = Tile::ptr(p.c, page, j, off >> 4);
#pragma unroll
  for (int pr = 0; pr < 2; ++pr) {
    const int g = HD == 128 ? pr : 0, i = HD == 128 ? l : pr * 16 + l;
    const float lo = g ? lo1 : lo0, hi = g ? hi1 : hi0;
    const __half sh = __float2half_rn(hi > lo ? __fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f) : 1.f), bh = __float2half_rn(lo);
    const float s = __half2float(sh), b = __half2float(bh);
    const unsigned byte = code4(x[2 * pr], s, b) | code4(x[2 * pr + 1], s, b) << 4;
    tile[is_v ? Tile::v_at(tt, g, i) : Tile::k_at(tt, g, i)] = static_cast<uint8_t>(byte);
    if (l == 0 && (HD == 128 || pr == 0))
      *reinterpret_cast<__half2*>(tile + Tile::kSb + tt * Tile::kEntry + (is_v ? 4 * Tile::G : 0) + 4 * g) =
          __halves2half2(sh, bh);
  }
}

// One thread per (token, KV head, K or V, byte pair of dims): two adjacent dims of one code byte.
template <int HD>
__global__ void __launch_bounds__(256) rows_kernel(Kv4 c, const int64_t* __restrict__ slots, int T,
                                                   __half* __restrict__ k, __half* __restrict__ v, unsigned* err) {
  using Tile = Kv4Tile<HD>;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t all = static_cast<int64_t>(T) * c.kvh * HD;  // (HD / 2) bytes x (K, V)
  if (i >= all) return;
  const int byte = static_cast<int>(i % (HD / 2)), is_v = static_cast<int>(i / (HD / 2) % 2);
  const int64_t th = i / HD;
  const int t = static_cast<int>(th / c.kvh), j = static_cast<int>(th % c.kvh);
  const int64_t slot = slots[t];
  __half2 out = __float2half2_rn(0.f);
  if (slot >= static_cast<int64_t>(c.pages) * c.page) {
    if (err) atomicOr(err, kErrBadPos);
  } else if (slot >= 0) {
    const int page = static_cast<int>(slot / c.page), off = static_cast<int>(slot % c.page), tt = off & 15;
    const uint8_t* tile = Tile::ptr(c, page, j, off >> 4);
    const int g = byte >> 5, b = byte & 31;
    const unsigned code = tile[is_v ? Tile::v_at(tt, g, b) : Tile::k_at(tt, g, b)];
    const float2 sb = __half22float2(*reinterpret_cast<const __half2*>(tile + Tile::kSb + tt * Tile::kEntry +
                                                                       (is_v ? 4 * Tile::G : 0) + 4 * g));
    out = __floats2half2_rn(__fmaf_rn(static_cast<float>(code & 15), sb.x, sb.y),
                            __fmaf_rn(static_cast<float>(code >> 4), sb.x, sb.y));
  }
  reinterpret_cast<__half2*>(is_v ? v : k)[th * (HD / 2) + byte] = out;
}

template <int HD>
int append_launch(const AppendParams& p, cudaStream_t s) {
  const int64_t items = static_cast<int64_t>(p.T) * (p.H + 2 * p.c.kvh);
  const int64_t grid = (items * (HD / 4) + 255) / 256;
  if (grid > 0x7fffffff) return fail(AGXC_EINVAL, "kv4_append: too many tokens for one call");
  const dim3 g(static_cast<unsigned>(grid));
  if (p.dtype == AGXC_F32) append_kernel<HD, AGXC_F32><<<g, 256, 0, s>>>(p);
  else if (p.dtype == AGXC_F16) append_kernel<HD, AGXC_F16><<<g, 256, 0, s>>>(p);
  else append_kernel<HD, AGXC_BF16><<<g, 256, 0, s>>>(p);
  AGXC_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace
}  // namespace agxc

using namespace agxc;

extern "C" {

AGXC_API int64_t agxc_kv4_bytes(const agxc_kv4_cache* c) {
  if (!c || (c->head_dim != 64 && c->head_dim != 128) || c->pages < 1 || c->kv_heads < 1 || c->page_size < 16 ||
      c->page_size % 16) {
    fail(AGXC_EINVAL, "kv4_bytes: head_dim 64 or 128, page_size a positive multiple of 16, pages and kv_heads >= 1");
    return -1;
  }
  const int64_t tile = c->head_dim == 128 ? Kv4Tile<128>::kBytes : Kv4Tile<64>::kBytes;
  return static_cast<int64_t>(c->pages) * c->kv_heads * (c->page_size / 16) * tile;
}

AGXC_API int agxc_kv4_append_dev(agxc_ctx* ctx, const agxc_kv4_append_args* a, void* stream) {
  if (!ctx || !a) return fail(AGXC_EINVAL, "kv4_append: null argument");
  if (int rc = kv4_check(&a->cache, "kv4_append")) return rc;
  if (a->tokens < 0) return fail(AGXC_EINVAL, "kv4_append: tokens >= 0");
  if (a->heads < 1 || a->heads % a->cache.kv_heads)
    return fail(AGXC_EINVAL, "kv4_append: heads a positive multiple of kv_heads");
  if (a->qkv_dtype < AGXC_F32 || a->qkv_dtype > AGXC_BF16)
    return fail(AGXC_EINVAL, "kv4_append: qkv fp32, fp16 or bf16");
  if (a->q_dtype != AGXC_F16 && a->q_dtype != AGXC_BF16) return fail(AGXC_EINVAL, "kv4_append: q fp16 or bf16");
  if (a->qkv_ld < static_cast<int64_t>(a->heads + 2 * a->cache.kv_heads) * a->cache.head_dim)
    return fail(AGXC_EINVAL, "kv4_append: qkv_ld < (heads + 2 kv_heads) head_dim");
  if (a->table_rows < 1) return fail(AGXC_EINVAL, "kv4_append: at least one row of the RoPE tables");
  if (!a->q_norm_dev != !a->k_norm_dev) return fail(AGXC_EINVAL, "kv4_append: q_norm and k_norm, or neither");
  if (a->tokens == 0) return 0;
  if (!a->qkv_dev || !a->positions_dev || !a->slots_dev || !a->cos_dev || !a->sin_dev || !a->q_dev)
    return fail(AGXC_EINVAL, "kv4_append: null buffer");
  AppendParams p;
  p.c = kv4_of(a->cache);
  p.qkv = a->qkv_dev; p.ld = a->qkv_ld; p.dtype = a->qkv_dtype; p.T = a->tokens; p.H = a->heads;
  p.table_rows = a->table_rows;
  p.pos = a->positions_dev; p.slots = a->slots_dev; p.cos_t = a->cos_dev; p.sin_t = a->sin_dev;
  p.bias = reinterpret_cast<const __half*>(a->bias_dev);
  p.qn = reinterpret_cast<const __half*>(a->q_norm_dev);
  p.kn = reinterpret_cast<const __half*>(a->k_norm_dev);
  p.eps = a->eps; p.qscale = a->qscale; p.q = a->q_dev; p.q_bf16 = a->q_dtype == AGXC_BF16; p.err = ctx->err_dev;
  cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  return a->cache.head_dim == 128 ? append_launch<128>(p, s) : append_launch<64>(p, s);
}

AGXC_API int agxc_kv4_rows_dev(agxc_ctx* ctx, const agxc_kv4_cache* cache, const int64_t* slots_dev, int tokens,
                               uint16_t* k_dev, uint16_t* v_dev, void* stream) {
  if (!ctx) return fail(AGXC_EINVAL, "kv4_rows: null context");
  if (int rc = kv4_check(cache, "kv4_rows")) return rc;
  if (tokens < 0) return fail(AGXC_EINVAL, "kv4_rows: tokens >= 0");
  if (tokens == 0) return 0;
  if (!slots_dev || !k_dev || !v_dev) return fail(AGXC_EINVAL, "kv4_rows: null buffer");
  cudaStream_t s = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
  const int64_t n = static_cast<int64_t>(tokens) * cache->kv_heads * cache->head_dim, grid = (n + 255) / 256;
  if (grid > 0x7fffffff) return fail(AGXC_EINVAL, "kv4_rows: too many tokens for one call");
  const dim3 g(static_cast<unsigned>(grid));
  __half* k = reinterpret_cast<__half*>(k_dev);
  __half* v = reinterpret_cast<__half*>(v_dev);
  if (cache->head_dim == 128) rows_kernel<128><<<g, 256, 0, s>>>(kv4_of(*cache), slots_dev, tokens, k, v, ctx->err_dev);
  else rows_kernel<64><<<g, 256, 0, s>>>(kv4_of(*cache), slots_dev, tokens, k, v, ctx->err_dev);
  AGXC_CUDA(cudaGetLastError());
  return 0;
}

}  // extern "C"
