// kv4.cu — the paged 4-bit KV cache's append and read-back (the attention over it is kv4_attention.cu).
//
//   append   x = qkv + bias; optional RMS norm of each q and k head; RoPE on (i, i + hd/2): o1 = x1 c - x2 s,
//            o2 = x2 c + x1 s, each product and sum rounded (as the fp16 cache's append); q = o * qscale, rounded;
//            k and v quantised per 64 dims: scale = (max - min) fp32(1 / 15) and bias = min in fp16 (scale 1 where all are
//            equal), code = rint((x - b) / s) clipped to 0..15, 0 where that is not finite; each step an IEEE fp32
//            operation, so the codes do not depend on how the tokens are batched. A NaN makes its group's bias NaN and with
//            it the whole group: the minimum and maximum keep it, where fminf and fmaxf would drop it and store a broken
//            value as the group's least.
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
  int q_bf16, vec;  // vec = every row, table and vector is aligned to four values
  unsigned* err;
};

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if (DT == AGXC_F32) return static_cast<const float*>(p)[i];
  if (DT == AGXC_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// four values from index i on, in one load where they are aligned to their size together
template <int DT>
__device__ __forceinline__ void load4(const void* p, int64_t i, bool vec, float* x) {
  if (!vec) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = load1<DT>(p, i + e);
    return;
  }
  if constexpr (DT == AGXC_F32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t h = ((e & 2 ? v.y : v.x) >> (16 * (e & 1))) & 0xffffu;
      x[e] = DT == AGXC_F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(h))) : __uint_as_float(h << 16);
    }
  }
}

// the smaller and the larger of two, NaN where either is
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// min and max over the LPH lanes of a head
template <int LPH>
__device__ __forceinline__ void head_minmax(float& lo, float& hi) {
#pragma unroll
  for (int m = LPH / 2; m >= 1; m >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
  }
}

__device__ __forceinline__ unsigned code4(float x, float s, float b) {
  const float q = rintf(__fdiv_rn(__fsub_rn(x, b), s));
  return isfinite(q) ? static_cast<unsigned>(fminf(fmaxf(q, 0.f), 15.f)) : 0u;
}

// hd / 8 lanes a head: lane l holds dims 4l .. 4l + 3 and the dims hd / 2 above them (four RoPE pairs, two code bytes
// side by side each). A warp takes two heads of 128 or four of 64.
// Every value is read once and each lane's loads, codes and q are one access each; 3,585 tokens of 14 + 2 x 2 heads of 64
// with the read back of their rows: 11.3 us (single values a lane took 14.0), where the bytes alone, 18.6 MB, take 2.8. The
// append's 2,017 CTAs of 40 registers are 2.3 waves of six an SM, and the issue slots are 65 of 100 taken: chains of load,
// exchange over the head's lanes, divide, store, the exchange run for the q heads too, which do not use it. One token: 3.5.
template <int HD, int DT>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
  using Tile = Kv4Tile<HD>;
  constexpr int LPH = HD / 8;
  pdl_enter(1);
  const unsigned heads = p.H + 2 * p.c.kvh, item = blockIdx.x * (256 / LPH) + threadIdx.x / LPH;
  const int l = threadIdx.x % LPH;
  const bool live = item < p.T * heads;
  const int t = live ? item / heads : 0, head = live ? item - t * heads : 0;
  const bool is_q = head < p.H, is_v = head >= p.H + p.c.kvh;
  float x[8];
  const int d0 = 4 * l, d1 = HD / 2 + 4 * l;
  const int64_t row = static_cast<int64_t>(t) * p.ld + head * HD;
  load4<DT>(p.qkv, row + d0, p.vec, x);
  load4<DT>(p.qkv, row + d1, p.vec, x + 4);
  const int pos = p.pos[t];
  const int64_t slot = p.slots[t];
  const bool bad = pos < 0 || pos >= p.table_rows || slot >= static_cast<int64_t>(p.c.pages) * p.c.page;
  if (live && bad && l == 0) atomicOr(p.err, kErrBadPos);
  float cs[4], sn[4];
  if (!is_v && !bad) {
    load4<AGXC_F32>(p.cos_t, static_cast<int64_t>(pos) * (HD / 2) + d0, p.vec, cs);
    load4<AGXC_F32>(p.sin_t, static_cast<int64_t>(pos) * (HD / 2) + d0, p.vec, sn);
  }
  if (p.bias) {
    float b[8];
    load4<AGXC_F16>(p.bias, head * HD + d0, p.vec, b);
    load4<AGXC_F16>(p.bias, head * HD + d1, p.vec, b + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(x[e], b[e]);
  }
  if (p.qn) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += x[e] * x[e];
#pragma unroll
    for (int m = LPH / 2; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (!is_v) {
      const float r = rsqrtf(sum / static_cast<float>(HD) + p.eps);
      const __half* g = is_q ? p.qn : p.kn;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (x[e] * r) * __half2float(g[e < 4 ? d0 + e : d1 + e - 4]);
    }
  }
  if (!is_v && !bad) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x1 = x[e], x2 = x[4 + e];
      x[e] = __fadd_rn(__fmul_rn(x1, cs[e]), -__fmul_rn(x2, sn[e]));
      x[4 + e] = __fadd_rn(__fmul_rn(x2, cs[e]), __fmul_rn(x1, sn[e]));
    }
  }
  // the shuffles below are the whole warp's
  float lo[2], hi[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    lo[h] = min_nan(min_nan(x[4 * h], x[4 * h + 1]), min_nan(x[4 * h + 2], x[4 * h + 3]));
    hi[h] = max_nan(max_nan(x[4 * h], x[4 * h + 1]), max_nan(x[4 * h + 2], x[4 * h + 3]));
  }
  if (HD == 64) {
    lo[0] = lo[1] = min_nan(lo[0], lo[1]);
    hi[0] = hi[1] = max_nan(hi[0], hi[1]);
  }
  head_minmax<LPH>(lo[0], hi[0]);
  if (HD == 128) head_minmax<LPH>(lo[1], hi[1]);
  if (!live || bad) return;
  if (is_q) {
    uint16_t* o = static_cast<uint16_t*>(p.q) + (static_cast<int64_t>(t) * p.H + head) * HD;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float a = __fmul_rn(x[4 * h + 2 * e], p.qscale), b = __fmul_rn(x[4 * h + 2 * e + 1], p.qscale);
        if (p.q_bf16) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
          w[e] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __half2 v = __floats2half2_rn(a, b);
          w[e] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      *reinterpret_cast<uint2*>(o + (h ? d1 : d0)) = make_uint2(w[0], w[1]);
    }
    return;
  }
  if (slot < 0) return;
  const int j = is_v ? head - p.H - p.c.kvh : head - p.H;
  const int page = static_cast<int>(quotient(slot, p.c.page));
  const int off = static_cast<int>(slot - static_cast<int64_t>(page) * p.c.page), tt = off & 15;
  uint8_t* tile = Tile::ptr(p.c, page, j, off >> 4);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int g = HD == 128 ? h : 0, i = HD == 128 ? 2 * l : h * 16 + 2 * l;
    const float low = HD == 128 ? lo[h] : lo[0], high = HD == 128 ? hi[h] : hi[0];
    const __half sh = __float2half_rn(high > low ? __fmul_rn(__fsub_rn(high, low), 1.f / 15.f) : 1.f);
    const __half bh = __float2half_rn(low);
    const float s = __half2float(sh), b = __half2float(bh);
    unsigned two = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) two |= code4(x[4 * h + e], s, b) << (4 * e);
    *reinterpret_cast<uint16_t*>(tile + (is_v ? Tile::v_at(tt, g, i) : Tile::k_at(tt, g, i))) = static_cast<uint16_t>(two);
    if (l == 0 && (HD == 128 || h == 0))
      *reinterpret_cast<__half2*>(tile + Tile::kSb + tt * Tile::kEntry + (is_v ? 4 * Tile::G : 0) + 4 * g) =
          __halves2half2(sh, bh);
  }
}

// One thread per (token, KV head, K or V, two bytes of codes): four adjacent dims.
template <int HD>
__global__ void __launch_bounds__(256) rows_kernel(Kv4 c, const int64_t* __restrict__ slots, int T,
                                                   __half* __restrict__ k, __half* __restrict__ v, unsigned* err) {
  using Tile = Kv4Tile<HD>;
  pdl_enter(1);
  const unsigned i = blockIdx.x * 256 + threadIdx.x, th = i / (HD / 2);  // hd / 4 threads each of K and V
  const int four = i % (HD / 4), is_v = i / (HD / 4) % 2, t = th / c.kvh, j = th - t * c.kvh;
  if (t >= T) return;
  const int64_t slot = slots[t];
  __half2 out[2] = {__float2half2_rn(0.f), __float2half2_rn(0.f)};
  if (slot >= static_cast<int64_t>(c.pages) * c.page) {
    atomicOr(err, kErrBadPos);
  } else if (slot >= 0) {
    const int page = static_cast<int>(quotient(slot, c.page));
    const int off = static_cast<int>(slot - static_cast<int64_t>(page) * c.page), tt = off & 15;
    const uint8_t* tile = Tile::ptr(c, page, j, off >> 4);
    const int g = four >> 4, b = 2 * (four & 15);
    const unsigned code = *reinterpret_cast<const uint16_t*>(tile + (is_v ? Tile::v_at(tt, g, b) : Tile::k_at(tt, g, b)));
    const float2 sb = __half22float2(*reinterpret_cast<const __half2*>(tile + Tile::kSb + tt * Tile::kEntry +
                                                                       (is_v ? 4 * Tile::G : 0) + 4 * g));
#pragma unroll
    for (int e = 0; e < 2; ++e)
      out[e] = __floats2half2_rn(__fmaf_rn(static_cast<float>(code >> (8 * e) & 15), sb.x, sb.y),
                                 __fmaf_rn(static_cast<float>(code >> (8 * e + 4) & 15), sb.x, sb.y));
  }
  uint2 w = make_uint2(*reinterpret_cast<uint32_t*>(&out[0]), *reinterpret_cast<uint32_t*>(&out[1]));
  *reinterpret_cast<uint2*>((is_v ? v : k) + static_cast<int64_t>(th) * HD + 4 * four) = w;
}

template <int HD>
int append_launch(const AppendParams& p, cudaStream_t s) {
  const int per = 256 / (HD / 8);
  const dim3 g(static_cast<unsigned>((static_cast<int64_t>(p.T) * (p.H + 2 * p.c.kvh) + per - 1) / per));
  if (p.dtype == AGXC_F32) return launch_ex(append_kernel<HD, AGXC_F32>, g, dim3(256), 0, s, 1, p);
  if (p.dtype == AGXC_F16) return launch_ex(append_kernel<HD, AGXC_F16>, g, dim3(256), 0, s, 1, p);
  return launch_ex(append_kernel<HD, AGXC_BF16>, g, dim3(256), 0, s, 1, p);
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
  if (reinterpret_cast<uintptr_t>(a->q_dev) % 8) return fail(AGXC_EINVAL, "kv4_append: q must be 8-byte aligned");
  if (static_cast<int64_t>(a->tokens) * (a->heads + 2 * a->cache.kv_heads) > 0x7fffffff)
    return fail(AGXC_EINVAL, "kv4_append: too many tokens for one call");
  const OnDevice on(ctx->device);
  if (on.rc()) return on.rc();
  AppendParams p;
  p.c = kv4_of(a->cache);
  p.qkv = a->qkv_dev; p.ld = a->qkv_ld; p.dtype = a->qkv_dtype; p.T = a->tokens; p.H = a->heads;
  p.table_rows = a->table_rows;
  p.pos = a->positions_dev; p.slots = a->slots_dev; p.cos_t = a->cos_dev; p.sin_t = a->sin_dev;
  p.bias = reinterpret_cast<const __half*>(a->bias_dev);
  p.qn = reinterpret_cast<const __half*>(a->q_norm_dev);
  p.kn = reinterpret_cast<const __half*>(a->k_norm_dev);
  p.eps = a->eps; p.qscale = a->qscale; p.q = a->q_dev; p.q_bf16 = a->q_dtype == AGXC_BF16; p.err = ctx->err_dev;
  const int size = a->qkv_dtype == AGXC_F32 ? 16 : 8;  // bytes of four values
  p.vec = reinterpret_cast<uintptr_t>(a->qkv_dev) % size == 0 && a->qkv_ld % 4 == 0 &&
          reinterpret_cast<uintptr_t>(a->cos_dev) % 16 == 0 && reinterpret_cast<uintptr_t>(a->sin_dev) % 16 == 0 &&
          reinterpret_cast<uintptr_t>(a->bias_dev) % 8 == 0;
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
  if (reinterpret_cast<uintptr_t>(k_dev) % 8 || reinterpret_cast<uintptr_t>(v_dev) % 8)
    return fail(AGXC_EINVAL, "kv4_rows: k and v must be 8-byte aligned");
  const int64_t n = static_cast<int64_t>(tokens) * cache->kv_heads * cache->head_dim / 2;
  if (n > 0x7fffffff - 256) return fail(AGXC_EINVAL, "kv4_rows: too many tokens for one call");
  const OnDevice on(ctx->device);
  if (on.rc()) return on.rc();
  const dim3 g(static_cast<unsigned>((n + 255) / 256));
  __half* k = reinterpret_cast<__half*>(k_dev);
  __half* v = reinterpret_cast<__half*>(v_dev);
  return cache->head_dim == 128
             ? launch_ex(rows_kernel<128>, g, dim3(256), 0, s, 1, kv4_of(*cache), slots_dev, tokens, k, v, ctx->err_dev)
             : launch_ex(rows_kernel<64>, g, dim3(256), 0, s, 1, kv4_of(*cache), slots_dev, tokens, k, v, ctx->err_dev);
}

}  // extern "C"
